"""MXFP4 (OCP microscaling: e2m1 elements, one power-of-two scale per 32 along the last dimension) on B200 through
libonebase_b200.so: quantization of weights and activations, and the values codes stand for.

codes [..., K/2] uint8 hold two elements per byte (element 2i in the low nibble), scales [..., K/32] uint8 exponent + 127 (255:
NaN) -- what VllmFusedMXFP4LoRA takes as its weight, and as its input under `quantized=`."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from onebase_b200 import _lib

BLOCK = 32
_DTYPE = {torch.bfloat16: _lib.OB_DTYPE_BF16, torch.float16: _lib.OB_DTYPE_F16, torch.float32: _lib.OB_DTYPE_F32}


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, shape, device) -> None:
    K = shape[-1]
    for name, t, want in (("codes", codes, (*shape[:-1], K // 2)), ("scales", scales, (*shape[:-1], K // BLOCK))):
        if t.dtype != torch.uint8 or tuple(t.shape) != tuple(want) or t.device != device or not t.is_contiguous():
            raise ValueError(f"mxfp4: {name} must be a dense uint8 tensor of shape {tuple(want)} on {device}")


def _rows(t: torch.Tensor):
    """(the tensor, rows, K, row pitch) as rows of the last dimension; a copy where its leading dimensions do not merge."""
    K = t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1:
        return t, t.shape[0], K, t.stride(0)
    t = t.reshape(-1, K)
    if t.stride(1) != 1:
        t = t.contiguous()
    return t, t.shape[0], K, t.stride(0)


def quantize(x: torch.Tensor, codes: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None):
    """x [..., K] (bf16, fp16 or fp32, K a multiple of 32) -> (codes, scales), written into the given tensors if any."""
    if x.device.type != "cuda":
        raise RuntimeError("onebase_b200 runs on CUDA devices only (there is no CPU path)")
    if x.dim() < 1 or x.dtype not in _DTYPE or x.shape[-1] < BLOCK or x.shape[-1] % BLOCK:
        raise ValueError("mxfp4.quantize: x must be bf16, fp16 or fp32 with a last dimension that is a multiple of 32")
    K = x.shape[-1]
    if codes is None:
        codes = torch.empty(*x.shape[:-1], K // 2, dtype=torch.uint8, device=x.device)
    if scales is None:
        scales = torch.empty(*x.shape[:-1], K // BLOCK, dtype=torch.uint8, device=x.device)
    _check_codes(codes, scales, x.shape, x.device)
    src, rows, K, ld = _rows(x)
    with torch.cuda.device(x.device):
        _lib.call("ob_mxfp4_quantize", C.c_void_p(src.data_ptr()), _DTYPE[x.dtype], rows, K, ld, C.c_void_p(codes.data_ptr()),
                  C.c_void_p(scales.data_ptr()), C.c_void_p(torch.cuda.current_stream(x.device).cuda_stream))
    return codes, scales


def dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values of codes [..., K/2] and scales [..., K/32] as `dtype` (exact in bf16 and fp32 while they are in its range)."""
    if codes.device.type != "cuda":
        raise RuntimeError("onebase_b200 runs on CUDA devices only (there is no CPU path)")
    if codes.dim() < 1 or codes.shape[-1] < BLOCK // 2 or codes.shape[-1] % (BLOCK // 2):
        raise ValueError("mxfp4.dequantize: codes must be [..., K/2] with K a multiple of 32")
    shape = (*codes.shape[:-1], 2 * codes.shape[-1])
    _check_codes(codes, scales, shape, codes.device)
    if out is None:
        if dtype not in _DTYPE:
            raise ValueError("mxfp4.dequantize: dtype must be bf16, fp16 or fp32")
        out = torch.empty(shape, dtype=dtype, device=codes.device)
    elif tuple(out.shape) != shape or out.dtype not in _DTYPE or out.device != codes.device or out.stride(-1) != 1 or \
            not (out.dim() == 2 or out.is_contiguous()):
        raise ValueError("mxfp4.dequantize: out must be bf16, fp16 or fp32 of the codes' shape and device, rows dense")
    dst = out if out.dim() == 2 else out.view(-1, shape[-1])
    with torch.cuda.device(codes.device):
        _lib.call("ob_mxfp4_dequantize", C.c_void_p(codes.data_ptr()), C.c_void_p(scales.data_ptr()), _DTYPE[out.dtype], dst.shape[0],
                  shape[-1], C.c_void_p(dst.data_ptr()), dst.stride(0), C.c_void_p(torch.cuda.current_stream(codes.device).cuda_stream))
    return out
