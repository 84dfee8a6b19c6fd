"""Microscaled 4-bit floating point (MXFP4): quantisation and products (``csrc/device/fp4_quant.cu``, ``fp4_gemm.cu``).

    w = quantize_fp4(weight)                    # once; or Fp4Tensor.from_parts(codes, scales) of a checkpoint
    y = gemm_fp4(quantize_fp4(x), w)            # x @ weight.T in 4 bits, fp32 accumulation, bf16 result

    recv = moe.dispatch(x, topk_idx)            # the experts' step between dispatch and combine
    h = gemm_fp4_swiglu(quantize_fp4(recv.rows, recv.scales, offsets=recv.expert_offsets), w_gate, w_up)
    y = gemm_fp4(quantize_fp4(h, offsets=recv.expert_offsets), w_down)

A value is e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives); every 32 consecutive ones of a row share a power of two, the
largest that keeps the block's largest magnitude at 4 or more before rounding (at least 2^-127).  Rounding is to the nearest, the even
one of two; magnitudes beyond 6 become 6.  A block that holds an infinity or a NaN becomes NaN.  None of these operators has a gradient.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from .. import _lib
from .._ext import Short
from .._stream import raw_stream

_TYPES = {torch.float32: _lib.FP32, torch.float16: _lib.FP16, torch.bfloat16: _lib.BF16, torch.float8_e4m3fn: _lib.FP8E4M3}
MAX_EXPERTS = 1024
_MOST = 2 ** 31 - 257          # rows, columns and depth of a product, which the library takes as 32-bit numbers


_short_quantize, _short_dequantize = Short("fp4_quantize", "HcommFp4Quantize"), Short("fp4_dequantize", "HcommFp4Dequantize")
_short_gemm, _short_swiglu = Short("fp4_gemm", "HcommFp4Gemm"), Short("fp4_gemm", "HcommFp4GemmSwiglu")


@dataclass(slots=True)
class Fp4Tensor:
    """A quantised matrix [rows, cols], or several of the same size [experts, rows, cols]."""
    values: torch.Tensor                    # uint8 [..., rows, cols // 2]: two values a byte, the even column in the low half
    scales: torch.Tensor                    # uint8 [tiles, 512]: exponents in tiles of 128 rows x 128 columns (include/hcomm_fp4.h)
    offsets: torch.Tensor | None = None     # int32 [experts + 1] on the device: rows grouped by expert

    @property
    def shape(self) -> tuple:
        return (*self.values.shape[:-1], 2 * self.values.shape[-1])

    @property
    def device(self) -> torch.device:
        return self.values.device

    @classmethod
    def from_parts(cls, values: torch.Tensor, scales: torch.Tensor) -> "Fp4Tensor":
        """Of what a checkpoint holds: values uint8 [..., rows, cols // 2], scales uint8 [..., rows, cols // 32] (biased exponents)."""
        if values.dtype != torch.uint8 or scales.dtype != torch.uint8 or values.dim() not in (2, 3):
            raise TypeError("values and scales must be uint8, values of two or three dimensions")
        if values.shape[:-1] != scales.shape[:-1] or values.shape[-1] != 16 * scales.shape[-1] or values.device != scales.device:
            raise ValueError(f"values {tuple(values.shape)} and scales {tuple(scales.shape)} do not belong together")
        *batch, rows, blocks = scales.shape
        s = scales.reshape(batch[0] if batch else 1, rows, blocks)          # in figures: -1 says nothing about an empty one
        if blocks % 4 or rows % 128:
            s = torch.nn.functional.pad(s, (0, -blocks % 4, 0, -rows % 128))
        s = s.view(s.shape[0], s.shape[1] // 128, 4, 32, s.shape[2] // 4, 4).permute(0, 1, 4, 3, 2, 5)
        values = values.contiguous()
        return cls(values if values.data_ptr() % 16 == 0 else values.clone(), s.reshape(s.shape[:3].numel(), 512).contiguous())

    def block_scales(self) -> torch.Tensor:
        """The scales as ``from_parts`` takes them, [..., rows, cols // 32]; not of grouped rows."""
        if self.offsets is not None:
            raise ValueError("rows grouped by expert have their scales in the experts' tiles")
        *batch, rows, cols = self.shape
        matrices, down, across = batch[0] if batch else 1, -(-rows // 128), -(-cols // 128)
        s = self.scales.view(matrices, down, across, 32, 4, 4).permute(0, 1, 4, 3, 2, 5)
        return s.reshape(matrices, down * 128, across * 4)[:, :rows, :cols // 32].reshape(*batch, rows, cols // 32)


def _on_device(what: str, *tensors) -> torch.device:
    device = tensors[0].device
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device != device):
            raise ValueError(f"{what} expects its tensors on one CUDA device, but got one on {t.device}")
    return device


def _pitch(dim: int, t: torch.Tensor) -> int:
    """Distance of neighbours along a dimension; of a dimension of one, whatever it says, its width."""
    return t.stride(dim) if t.shape[dim] > 1 else max(t.stride(dim), t.shape[-1])


def _check_offsets(offsets):
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or not offsets.is_contiguous() or not 2 <= offsets.shape[0] <= MAX_EXPERTS + 1:
        raise ValueError(f"offsets must be a contiguous int32 vector of 2 to {MAX_EXPERTS + 1} entries")


def _call(name: str, device: torch.device, *args):
    if torch.cuda.current_device() == device.index:
        rc = getattr(_lib.load(), name)(*args)
    else:
        with torch.cuda.device(device):
            rc = getattr(_lib.load(), name)(*args)
    if rc:
        _lib.check(rc, name)


def _ptr(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr() if t is not None else None)


_i64 = ctypes.c_int64


def _scale_tiles(batch: int, rows: int, cols: int, experts: int) -> int:
    """Tiles of scales (``HcommFp4ScaleBytes`` / 512)."""
    tile_rows = rows // 128 + min(rows, experts) if experts else batch * -(-rows // 128)
    return tile_rows * -(-cols // 128)


def quantize_fp4(x: torch.Tensor, scales: torch.Tensor | None = None, *, offsets: torch.Tensor | None = None) -> Fp4Tensor:
    """x [rows, cols] or [experts, rows, cols] in fp32, fp16 or bf16, cols a multiple of 32, the last dimension contiguous.

    With ``scales`` [rows, cols // 128] (fp32), x [rows, cols] is fp8 e4m3 and stands for the products with its scales, as rows
    that the expert-parallel exchange delivers; cols a multiple of 128.  With ``offsets`` (int32 [experts + 1]) rows
    offsets[e] .. offsets[e + 1] belong to expert e: the result is the left operand of a product with every expert's own matrix.
    Rows behind the last expert's are neither read nor written."""
    r = _short_quantize(x, scales, offsets)
    if r is not None:
        return Fp4Tensor(r[0], r[1], offsets)
    device = _on_device("quantize_fp4", x, scales, offsets)
    fp8 = x.dtype == torch.float8_e4m3fn
    if x.dtype not in _TYPES or fp8 != (scales is not None):
        raise TypeError("quantize_fp4 takes fp32, fp16 or bf16, or float8_e4m3fn with its scales")
    if x.dim() not in (2, 3) or (x.dim() == 3 and (fp8 or offsets is not None)):
        raise ValueError("x must be [rows, cols], or [experts, rows, cols] without scales and offsets")
    rows, cols = x.shape[-2:]
    batch = x.shape[0] if x.dim() == 3 else 1
    if cols % (128 if fp8 else 32):
        raise ValueError(f"{cols} columns: a multiple of {128 if fp8 else 32} is needed")
    if x.numel() and cols > 1 and x.stride(-1) != 1:
        raise ValueError("the last dimension must be contiguous")
    scale_pitch = 0
    if fp8:
        if scales.dtype != torch.float32 or tuple(scales.shape) != (rows, cols // 128):
            raise ValueError(f"scales must be fp32 [{rows}, {cols // 128}]")
        if scales.numel() and scales.shape[1] > 1 and scales.stride(1) != 1:
            raise ValueError("the last dimension of the scales must be contiguous")
        scale_pitch = _pitch(0, scales)
    experts = 0
    if offsets is not None:
        _check_offsets(offsets)
        experts = offsets.shape[0] - 1
    values = torch.empty((*x.shape[:-1], cols // 2), dtype=torch.uint8, device=device)
    tiles = torch.empty((_scale_tiles(batch, rows, cols, experts), 512), dtype=torch.uint8, device=device)
    if x.numel():
        _call("HcommFp4Quantize", device, _ptr(x), _TYPES[x.dtype], _ptr(scales), _i64(batch), _i64(rows), _i64(cols), _i64(_pitch(0, x) if x.dim() == 3 else 0),
              _i64(_pitch(-2, x)), _i64(scale_pitch), _ptr(offsets), experts, _ptr(values), _ptr(tiles), ctypes.c_void_p(raw_stream(x)))
    return Fp4Tensor(values, tiles, offsets)


def dequantize_fp4(q: Fp4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that q stands for, in bf16 (exact unless tiny), fp16 or fp32.  Rows behind the last expert's are left undefined."""
    r = _short_dequantize(q.values, q.scales, q.offsets, _TYPES.get(dtype, -1)) if q.__class__ is Fp4Tensor else None
    if r is not None:
        return r
    device = _check_operand("dequantize_fp4", q)
    if dtype not in _TYPES or dtype == torch.float8_e4m3fn:
        raise TypeError("dequantize_fp4 makes fp32, fp16 or bf16")
    *batch, rows, cols = q.shape
    out = torch.empty(q.shape, dtype=dtype, device=device)
    if out.numel():
        _call("HcommFp4Dequantize", device, _ptr(q.values), _ptr(q.scales), _i64(batch[0] if batch else 1), _i64(rows), _i64(cols), _ptr(q.offsets),
              q.offsets.shape[0] - 1 if q.offsets is not None else 0, _ptr(out), _TYPES[dtype], ctypes.c_void_p(raw_stream(out)))
    return out


def _check_operand(what: str, q: Fp4Tensor) -> torch.device:
    if not isinstance(q, Fp4Tensor):
        raise TypeError(f"{what} expects an Fp4Tensor")
    device = _on_device(what, q.values, q.scales, q.offsets)
    if q.values.dtype != torch.uint8 or q.scales.dtype != torch.uint8 or q.values.dim() not in (2, 3) or not q.values.is_contiguous() or not q.scales.is_contiguous():
        raise ValueError("values and scales must be contiguous uint8, values of two or three dimensions")
    experts = 0
    if q.offsets is not None:
        _check_offsets(q.offsets)
        experts = q.offsets.shape[0] - 1
        if q.values.dim() != 2:
            raise ValueError("rows grouped by expert are one matrix")
    *batch, rows, cols = q.shape
    if cols % 32 or q.scales.numel() != 512 * _scale_tiles(batch[0] if batch else 1, rows, cols, experts):
        raise ValueError(f"{q.scales.numel()} bytes of scales do not belong to {tuple(q.shape)}")
    return device


def _result(what: str, a: Fp4Tensor, weights, out):
    device = _check_operand(what, a)
    shape = weights[0].shape
    for w in weights:
        if _check_operand(what, w) != device:
            raise ValueError(f"{what} expects its operands on one device")
        if w.offsets is not None or w.shape != shape:
            raise ValueError("weights must have the same shape and no groups of rows")
    if len(a.shape) != 2 or a.shape[1] != shape[-1] or len(shape) != (2 if a.offsets is None else 3):
        raise ValueError(f"shapes {tuple(a.shape)} x {tuple(shape)}^T do not match; rows grouped by expert take a matrix for each expert, other rows take one")
    if a.offsets is not None and a.offsets.shape[0] - 1 != shape[0]:
        raise ValueError(f"{a.offsets.shape[0] - 1} groups of rows for {shape[0]} experts")
    if shape[-1] == 0:
        raise ValueError("no columns to multiply")
    m, n = a.shape[0], shape[-2]
    if max(m, n, shape[-1]) > _MOST:
        raise ValueError(f"a product of {m} x {n} x {shape[-1]}: at most {_MOST} of each")
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=device)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (m, n) or out.device != device:
        raise ValueError(f"out must be bfloat16 [{m}, {n}] on {device}")
    elif out.numel() and ((n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n)):
        raise ValueError("rows of out must be contiguous and not overlap")
    return out, device, m, n


def _multiply(name: str, what: str, a: Fp4Tensor, weights, out):
    out, device, m, n = _result(what, a, weights, out)
    if m and n:
        operands = [_ptr(t) for q in (a, *weights) for t in (q.values, q.scales)]
        _call(name, device, *operands, _ptr(out), m, n, a.shape[1], _i64(_pitch(0, out)), _ptr(a.offsets), a.offsets.shape[0] - 1 if a.offsets is not None else 0,
              ctypes.c_void_p(raw_stream(out)))
    return out


def gemm_fp4(a: Fp4Tensor, b: Fp4Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``a @ b.T`` of a [M, K] and b [N, K], bf16 [M, N].

    Of rows grouped by expert and b [experts, N, K], each row with its expert's matrix; rows of ``out`` behind the last expert's are
    left as they were."""
    if a.__class__ is Fp4Tensor and b.__class__ is Fp4Tensor and b.offsets is None:
        r = _short_gemm(a.values, a.scales, a.offsets, out, b.values, b.scales)
        if r is not None:
            return r
    return _multiply("HcommFp4Gemm", "gemm_fp4", a, (b,), out)


def gemm_fp4_swiglu(a: Fp4Tensor, gate: Fp4Tensor, up: Fp4Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(a @ gate.T) * (a @ up.T)``, bf16, from the fp32 accumulators of both; rows grouped by expert as in ``gemm_fp4``.

    silu is taken as 0 where its argument is below -87.3, where its magnitude is below 2^-119."""
    if a.__class__ is gate.__class__ is up.__class__ is Fp4Tensor and gate.offsets is up.offsets is None:
        r = _short_swiglu(a.values, a.scales, a.offsets, out, gate.values, gate.scales, up.values, up.scales)
        if r is not None:
            return r
    return _multiply("HcommFp4GemmSwiglu", "gemm_fp4_swiglu", a, (gate, up), out)


def take_kernel_error() -> int:
    """Non-zero when a bounded wait inside a 4-bit product expired since the last call (clears the flag)."""
    return int(_lib.load().HcommFp4TakeError())
