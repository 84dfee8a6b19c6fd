"""Expert-parallel feed-forward layer: routing, exchange, the experts in 4 bits, and the weighted sum back.

Every rank holds ``experts / comm.size`` experts and some tokens.  A forward pass is nine kernels on one rank (the router's product,
routing, dispatch, quantisation, gate and up products, quantisation, down product, sum; two for routing beyond 32 tokens) and never waits for the GPU: how many rows an
expert gets is known on the device only.
"""
from __future__ import annotations

import torch

from ..comm import Communicator
from ..ops.fp4 import Fp4Tensor, gemm_fp4, gemm_fp4_swiglu, quantize_fp4
from ..ops.gemm import gemm_bf16
from ..ops.moe import MoeExchange
from ..ops.router import route


class ExpertParallelMlp:
    """``combine(gates, down_e(silu(gate_e(x)) * up_e(x)))`` over the ``topk`` experts e of each token; inference only.

    The router's logits are products in bf16 with fp32 sums, rounded to bf16 as ``gemm_bf16`` leaves them: experts whose logits agree in those eight
    bits are a tie, which the lower index wins.  A program that routes on logits in fp32 calls ``route`` and the exchange itself.
    Products by expert are planned for the rows that ``max_tokens`` may bring, so a layer made for what a step holds is the faster one.

    Weights: router bf16 [experts, hidden]; gate and up [local experts, intermediate, hidden] and down [local experts, hidden,
    intermediate], bf16 (quantised here) or ``Fp4Tensor``; random-initialised N(0, 0.02) unless given.  hidden as ``MoeExchange`` takes it,
    intermediate a multiple of 32.  Creating a layer is a collective call, and so is each forward pass; passes of one layer
    follow one another on a stream (they share its buffers)."""

    def __init__(self, comm: Communicator, experts: int, topk: int, hidden: int, intermediate: int, max_tokens: int, device=None, seed: int = 0, w_router=None, w_gate=None,
                 w_up=None, w_down=None, scoring: str = "softmax", renormalize: bool = True, scale: float = 1.0, bias: torch.Tensor | None = None, capacity_factor: float = 2.0):
        dev = device or torch.device("cuda", torch.cuda.current_device())
        if experts % 8:
            raise ValueError(f"{experts} experts: a multiple of 8 is needed for the router's product")
        local = experts // comm.size
        shared = torch.Generator(device=dev).manual_seed(seed)                          # the same router on every rank
        own = torch.Generator(device=dev).manual_seed(seed + 1000 * (comm.rank + 1))

        def weight(given, shape, g, four_bits=True):
            if given is None:
                given = (torch.randn(shape, device=dev, generator=g) * 0.02).to(torch.bfloat16)
            if tuple(given.shape) != shape:
                raise ValueError(f"weights of {tuple(given.shape)} where {shape} are needed")
            return quantize_fp4(given) if four_bits and not isinstance(given, Fp4Tensor) else given
        self.router = weight(w_router, (experts, hidden), shared, four_bits=False)
        self.gate = weight(w_gate, (local, intermediate, hidden), own)
        self.up = weight(w_up, (local, intermediate, hidden), own)
        self.down = weight(w_down, (local, hidden, intermediate), own)
        self.topk, self.options = topk, dict(scoring=scoring, renormalize=renormalize, scale=scale, bias=bias)
        self.moe = MoeExchange(comm, experts, topk, hidden, max_tokens, capacity_factor)
        rows = self.moe.layout.maxRecvRows
        # what lies behind a step's last row is not read, but 0 and not whatever the memory held before
        self._h = torch.zeros((rows, intermediate), dtype=torch.bfloat16, device=dev)
        self._y = torch.zeros((rows, hidden), dtype=torch.bfloat16, device=dev)

    def forward(self, x: torch.Tensor, out: torch.Tensor | None = None, valid: torch.Tensor | None = None) -> torch.Tensor:
        """x [tokens, hidden] bf16; tokens that ``valid`` (bool [tokens]) takes out go to no expert and come back as 0.  A rank without
        tokens takes part all the same, as the pass is collective: with one that is taken out."""
        self._check(x, out)
        if x.shape[0] == 0:
            self.forward(x.new_zeros((1, x.shape[1])), valid=torch.zeros(1, dtype=torch.bool, device=x.device))
            return torch.empty_like(x) if out is None else out
        r = self.routing = route(gemm_bf16(x, self.router), self.topk, valid=valid, **self.options)
        recv = self.moe.dispatch(x, r.topk_idx)
        offsets = recv.expert_offsets
        h = gemm_fp4_swiglu(quantize_fp4(recv.rows, recv.scales, offsets=offsets), self.gate, self.up, self._h)
        y = gemm_fp4(quantize_fp4(h, offsets=offsets), self.down, self._y)
        return self.moe.combine(y, r.gates, out, nan_gates=True)

    __call__ = forward

    def _check(self, x, out):
        """Before anything is queued: the exchange behind is a collective call, and writes where it is told to."""
        shape, device, kind = x.shape, x.device, torch.bfloat16
        if len(shape) != 2 or shape[1] != self.moe.hidden or x.dtype is not kind or not x.is_contiguous() or device != self.router.device:
            raise ValueError(f"x must be contiguous bfloat16 [tokens, {self.moe.hidden}] on {self.router.device}")
        if shape[0] > self.moe.max_tokens:
            raise ValueError(f"{shape[0]} tokens: the layer was made for {self.moe.max_tokens}")
        if out is not None and (out.dtype is not kind or out.dim() != 2 or out.shape[0] < shape[0] or out.shape[1] != shape[1] or not out.is_contiguous() or out.device != device):
            raise ValueError(f"out must be contiguous bfloat16 {list(shape)} on {device}, or have more rows, which are left as they are")

    def destroy(self):
        self.moe.destroy()
