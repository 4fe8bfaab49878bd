"""MXFP4 (OCP microscaling: e2m1 elements, one power-of-two scale per 32 along the last dimension) on B200 through
libonebase_b200.so: quantization of weights and activations, and the values codes stand for.

codes [..., K/2] uint8 hold two elements per byte (element 2i in the low nibble), scales [..., K/32] uint8 exponent + 127 (255:
NaN) -- what VllmFusedMXFP4LoRA takes as its weight, and as its input under `quantized=`."""
from __future__ import annotations

from typing import Optional

import torch

from onebase_b200 import _lib

BLOCK = 32
_DTYPE = {torch.bfloat16: _lib.OB_DTYPE_BF16, torch.float16: _lib.OB_DTYPE_F16, torch.float32: _lib.OB_DTYPE_F32}


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, shape, device) -> None:
    K = shape[-1]
    for t, want in ((codes, (*shape[:-1], K // 2)), (scales, (*shape[:-1], K // BLOCK))):
        if t.dtype != torch.uint8 or t.shape != want or t.device != device or not t.is_contiguous():
            raise ValueError(f"mxfp4: codes and scales must be dense uint8 tensors, here one of shape {tuple(want)} on {device}")


def quantize(x: torch.Tensor, codes: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None):
    """x [..., K] (bf16, fp16 or fp32, K a multiple of 32) -> (codes, scales), written into the given tensors if any (which may be a
    projection's weight: the next call sees it)."""
    if not x.is_cuda:
        raise RuntimeError("onebase_b200 runs on CUDA devices only (there is no CPU path)")
    shape = x.shape
    if not shape or x.dtype not in _DTYPE or shape[-1] < BLOCK or shape[-1] % BLOCK:
        raise ValueError("mxfp4.quantize: x must be bf16, fp16 or fp32 with a last dimension that is a multiple of 32")
    K = shape[-1]
    given = codes is not None or scales is not None
    if codes is None:
        codes = x.new_empty((*shape[:-1], K // 2), dtype=torch.uint8)
    if scales is None:
        scales = x.new_empty((*shape[:-1], K // BLOCK), dtype=torch.uint8)
    if given:
        _check_codes(codes, scales, shape, x.device)
    src, st = x, x.stride()
    if len(st) != 2 or st[1] != 1:               # rows of the last dimension; a copy where the leading dimensions do not merge
        src = x.reshape(-1, K)
        if src.stride(1) != 1:
            src = src.contiguous()
        shape, st = src.shape, src.stride()
    _lib.call_on(x.device, "ob_mxfp4_quantize", src.data_ptr(), _DTYPE[x.dtype], shape[0], K, st[0], codes.data_ptr(),
                 scales.data_ptr())
    if given:
        _lib.call_on(x.device, "ob_operand_fence")
    return codes, scales


def dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values of codes [..., K/2] and scales [..., K/32] as `dtype` (exact in bf16 and fp32 while they are in its range), written
    into `out` if given (which may be a projection's adapter: the next call sees it)."""
    if not codes.is_cuda:
        raise RuntimeError("onebase_b200 runs on CUDA devices only (there is no CPU path)")
    if codes.dim() < 1 or codes.shape[-1] < BLOCK // 2 or codes.shape[-1] % (BLOCK // 2):
        raise ValueError("mxfp4.dequantize: codes must be [..., K/2] with K a multiple of 32")
    K = 2 * codes.shape[-1]
    shape = (*codes.shape[:-1], K)
    _check_codes(codes, scales, shape, codes.device)
    given = out is not None
    if not given:
        if dtype not in _DTYPE:
            raise ValueError("mxfp4.dequantize: dtype must be bf16, fp16 or fp32")
        out = codes.new_empty(shape, dtype=dtype)
    elif out.shape != shape or out.dtype not in _DTYPE or out.device != codes.device or out.stride(-1) != 1 or \
            not (out.dim() == 2 or out.is_contiguous()):
        raise ValueError("mxfp4.dequantize: out must be bf16, fp16 or fp32 of the codes' shape and device, rows dense")
    dst = out if out.dim() == 2 else out.view(-1, K)
    _lib.call_on(codes.device, "ob_mxfp4_dequantize", codes.data_ptr(), scales.data_ptr(), _DTYPE[out.dtype], dst.shape[0], K,
                 dst.data_ptr(), dst.stride(0))
    if given:
        _lib.call_on(codes.device, "ob_operand_fence")
    return out
