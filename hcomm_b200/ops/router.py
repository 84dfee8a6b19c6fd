"""Top-k routing with per-expert counts and a balance loss (``csrc/device/router_kernels.cu``): what ``MoeExchange`` takes.

    r = route(x @ w_router.T, topk=8, balance=0.01)         # logits [T, experts]
    recv = moe.dispatch(x, r.topk_idx)
    ... the experts ...
    out = moe.combine(y, r.gates, nan_gates=True)
    loss = task_loss + r.loss

``gates`` and ``loss`` have gradients with regard to the logits (in reverse mode, once); choices and counts are constants.  With f_e the share of the
tokens' choices that went to expert e and P_e the tokens' mean probability of it, the loss is ``balance * experts * sum f_e P_e``, which is
``balance`` where both are even.  A backward pass is captured into a CUDA graph while no eager graph of the same leaves lives, which is torch's rule for
every operator.
"""
from __future__ import annotations

import ctypes
import operator
from typing import NamedTuple

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from .. import _lib
from .._ext import Short, entry
from .._stream import raw_stream
from ..comm import Communicator

SCORINGS = {"softmax": 0, "sigmoid": 1}
_TYPES = {torch.float32: _lib.FP32, torch.float16: _lib.FP16, torch.bfloat16: _lib.BF16}
MAX_EXPERTS, MAX_TOPK = 1024, 16
_MOST_TOKENS = 2 ** 31 - 33           # the library counts them in 32 bits


class _ShortRoute(Short):
    """The native call, which is given the entry points of the backward pass and of the scratch's size as well."""

    __slots__ = ("_others",)

    def find(self):
        self._others = entry("HcommMoeRouteBackward"), entry("HcommMoeRouteScratchBytes")      # before another thread can see the call
        return super().find()

    def __call__(self, *args):
        if self._call is None:
            self.find()
        return super().__call__(*self._others, *args)


_short_route = _ShortRoute("moe_route", "HcommMoeRoute")


class Routing(NamedTuple):
    topk_idx: torch.Tensor          # int32 [T, topk]: experts, the best first; -1 where the token has nothing (more) to choose
    gates: torch.Tensor             # float32 [T, topk], 0 where topk_idx is -1
    counts: torch.Tensor            # int32 [experts]: tokens that chose each expert
    loss: torch.Tensor | None       # float32 scalar, None without a balance coefficient


_ptr, _f32, _i64 = ctypes.c_void_p, ctypes.c_float, ctypes.c_int64


def _address(t):
    return _ptr(None if t is None else t.data_ptr())


def _call(name: str, device: torch.device, *args):
    if torch.cuda.current_device() == device.index:
        rc = getattr(_lib.load(), name)(*args)
    else:
        with torch.cuda.device(device):
            rc = getattr(_lib.load(), name)(*args)
    if rc:
        _lib.check(rc, name)


def _pitch(logits):
    return _i64(logits.stride(0) if logits.shape[0] > 1 else max(logits.stride(0), logits.shape[1]))


def _scratch_bytes(tokens: int, experts: int) -> int:
    size = _lib.load().HcommMoeRouteScratchBytes
    size.restype = ctypes.c_uint64
    return size(tokens, experts)


def _forward(logits, topk, scoring, renormalize, scale, bias, valid, balance, comm):
    """topk_idx, gates, counts with the number of tokens behind them, loss."""
    t, e = logits.shape
    device = logits.device
    idx = torch.empty((t, topk), dtype=torch.int32, device=device)
    gates = torch.empty((t, topk), dtype=torch.float32, device=device)
    counts = torch.empty(e + 1, dtype=torch.int32, device=device)
    loss = torch.empty((), dtype=torch.float32, device=device) if balance else None
    sums = torch.empty(e, dtype=torch.float32, device=device) if balance and comm is not None else None
    scratch = torch.empty(_scratch_bytes(t, e), dtype=torch.uint8, device=device)
    stream = _ptr(raw_stream(logits))
    _call("HcommMoeRoute", device, _address(logits), _TYPES[logits.dtype], _pitch(logits), t, e, topk, scoring, int(renormalize), _f32(scale), _address(bias), _address(valid),
          _address(idx), _address(gates), _address(counts), _address(sums), _f32(balance), _address(loss if sums is None else None), _address(scratch), stream)
    if comm is not None:
        counts = comm.all_reduce(counts, torch.empty_like(counts))
        if balance:
            sums = comm.all_reduce(sums, torch.empty_like(sums))
            _call("HcommMoeBalanceLoss", device, _address(counts), _address(sums), e, topk, _f32(balance), _address(loss), stream)
    return idx, gates, counts, loss


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, scoring, renormalize, scale, bias, valid, balance, comm):
        idx, gates, counts, loss = _forward(logits, topk, scoring, renormalize, scale, bias, valid, balance, comm)
        ctx.save_for_backward(logits, valid, idx, counts)
        ctx.settings = scoring, renormalize, scale, balance
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(idx, counts)
        return idx, gates, counts, loss

    @staticmethod
    @once_differentiable
    def backward(ctx, _idx, dgates, _counts, dloss):
        none = (None,) * 8
        if dgates is None and dloss is None:
            return None, *none
        logits, valid, idx, counts = ctx.saved_tensors
        scoring, renormalize, scale, balance = ctx.settings
        if dgates is not None:
            dgates = dgates.contiguous()
        t, e = logits.shape
        grad = torch.empty((t, e), dtype=logits.dtype, device=logits.device)
        if t:
            _call("HcommMoeRouteBackward", logits.device, _address(logits), _TYPES[logits.dtype], _pitch(logits), t, e, idx.shape[1], scoring, int(renormalize), _f32(scale),
                  _address(valid), _address(idx), _address(dgates), _address(counts), _f32(balance), _address(dloss), _address(grad), _i64(e), _ptr(raw_stream(logits)))
        return grad, *none


def route(logits: torch.Tensor, topk: int, *, scoring: str = "softmax", renormalize: bool = True, scale: float = 1.0, bias: torch.Tensor | None = None,
          valid: torch.Tensor | None = None, balance: float = 0.0, comm: Communicator | None = None) -> Routing:
    """logits [T, experts] in fp32, fp16 or bf16, the last dimension contiguous; up to 1024 experts, topk up to 16.

    scoring      "softmax" over the experts or "sigmoid" of each; gates are the scores of the choices, with ``renormalize`` divided
                 by their sum over the token's choices, times ``scale``
    bias         float32 [experts], sigmoid only: added to the scores for the choice, not for the gates (no gradient)
    valid        bool [T]: tokens that are padding choose -1, have gates of 0, and count neither in ``counts`` nor in the loss
    balance      coefficient of the loss; 0: none is computed
    comm         counts and loss over the tokens of all ranks of a communicator (a collective call); each rank's gradient is that of
                 the one loss with regard to its own logits

    A logit of -inf takes the expert out for the token.  A row that holds a NaN (under softmax: or +inf) chooses -1 with gates of NaN,
    which ``MoeExchange.combine(..., nan_gates=True)`` carries on."""
    if comm is None and topk.__class__ is int and scoring in SCORINGS:
        r = _short_route(logits, topk, SCORINGS[scoring], 1 if renormalize else 0, float(scale), bias, valid, float(balance))
        if r is not None:
            return Routing(*r)
    if scoring not in SCORINGS:
        raise ValueError(f"scoring must be one of {sorted(SCORINGS)}")
    if logits.dim() != 2 or logits.dtype not in _TYPES:
        raise TypeError("logits must be [T, experts] in fp32, fp16 or bf16")
    t, e = logits.shape
    topk = operator.index(topk)
    if not 1 <= e <= MAX_EXPERTS or not 1 <= topk <= min(e, MAX_TOPK):
        raise ValueError(f"{topk} of {e} experts: at least one and at most {MAX_TOPK} of at most {MAX_EXPERTS}")
    if t > _MOST_TOKENS:
        raise ValueError(f"{t} tokens: at most {_MOST_TOKENS}")
    if not logits.is_cuda:
        raise ValueError(f"expected a tensor on a CUDA device, but got one on {logits.device}")
    if (e > 1 and logits.stride(1) != 1) or (t > 1 and logits.stride(0) < e):
        raise ValueError("the last dimension must be contiguous and rows may not overlap")
    if bias is not None:
        if scoring != "sigmoid":
            raise ValueError("a selection bias goes with sigmoid scores")
        if bias.dtype != torch.float32 or bias.shape != (e,) or bias.device != logits.device:
            raise ValueError(f"bias must be float32 [{e}] on {logits.device}")
        bias = bias.detach().contiguous()
    if valid is not None:
        if valid.dtype != torch.bool or valid.shape != (t,) or valid.device != logits.device:
            raise ValueError(f"valid must be bool [{t}] on {logits.device}")
        valid = valid.contiguous()
    args = (logits, topk, SCORINGS[scoring], bool(renormalize), float(scale), bias, valid, float(balance), comm)
    # a tangent of forward mode goes to the function as well, which has none to offer and says so
    followed = (logits.requires_grad and torch.is_grad_enabled()) or unpack_dual(logits).tangent is not None
    idx, gates, counts, loss = _Route.apply(*args) if followed else _forward(*args)
    return Routing(idx, gates, counts[:e], loss)
