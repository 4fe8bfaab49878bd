"""Root-mean-square norm with the residual's addition before it and low-precision codes behind it, on B200 through
libonebase_b200.so (ob_rms_norm).

In a decoder layer it stands in front of qkv_proj and gate_up_proj and gives a fused projection its input together with the
codes the projection multiplies:

    n = rms_norm(x, weight, eps, residual=stream, quant="fp8")
    y = op(n.y, meta, quantized=(n.codes, n.scales))        # VllmFusedFP8LoRA; quant="mxfp4" for VllmFusedMXFP4LoRA

and, on [tokens, heads, head size], it is the norm of queries and keys.  The reference leaves the norm to vLLM (RMSNorm,
vllm/model_executor/layers/layernorm.py).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from onebase_b200 import _lib

_ROWS = {torch.bfloat16: _lib.OB_DTYPE_BF16, torch.float16: _lib.OB_DTYPE_F16}
_WEIGHT = {**_ROWS, torch.float32: _lib.OB_DTYPE_F32}
_QUANT = {None: _lib.OB_QUANT_NONE, "fp8": _lib.OB_QUANT_FP8, "mxfp4": _lib.OB_QUANT_MXFP4}


class NormOut(NamedTuple):
    y: Optional[torch.Tensor]          # the norm, dtype of x (None under store=False)
    residual: Optional[torch.Tensor]   # x + residual, dtype of x (None without a residual)
    codes: Optional[torch.Tensor]      # "fp8": float8_e4m3fn, shape of x; "mxfp4": packed e2m1 uint8 [..., K/2]
    scales: Optional[torch.Tensor]     # "fp8": fp32 [...]; "mxfp4": exponent + 127, uint8 [..., K/32]


_NO_ROWS = (None, 0, 0)


def _rows(t: torch.Tensor, dims: int):
    """(pointer, stride between tokens, between heads)."""
    st = t.stride()
    return t.data_ptr(), st[0], st[1] if dims == 3 else 0


def _like(name: str, t: torch.Tensor, shape, dtype, device) -> None:
    if t.shape != shape or t.dtype != dtype or t.device != device or (t.stride(-1) != 1 and shape[-1] > 1):
        raise ValueError(f"rms_norm: {name} must have x's shape, dtype and device, its last dimension dense")


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-6, *, residual: Optional[torch.Tensor] = None,
             residual_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, store: bool = True,
             quant: Optional[str] = None) -> NormOut:
    """x [M, K] or [M, H, K] (bf16 or fp16, the last dimension dense, any other strides); weight [K] of x's dtype or fp32, or
    None; residual of x's shape and dtype: s = x + residual is returned (in residual_out if given: it may be the residual
    itself) and s is what is normed.  y = (s * weight) / sqrt(mean(s^2) + eps) goes to `out` (it may be x), or nowhere with
    store=False.  quant = "fp8" or "mxfp4" also returns the codes of y before its rounding to 16 bits, with their scales."""
    if not x.is_cuda:
        raise RuntimeError("onebase_b200 runs on CUDA devices only (there is no CPU path)")
    shape, dims, dtype, device = x.shape, x.dim(), x.dtype, x.device
    if dims not in (2, 3) or dtype not in _ROWS or shape[-1] < 1 or (x.stride(-1) != 1 and shape[-1] > 1):
        raise ValueError("rms_norm: x must be [M, K] or [M, H, K], bf16 or fp16, its last dimension dense")
    if quant not in _QUANT:
        raise ValueError("rms_norm: quant must be None, 'fp8' or 'mxfp4'")
    K = shape[-1]
    H = shape[1] if dims == 3 else 1
    if H < 1:
        raise ValueError("rms_norm: x has no heads")
    if weight is not None and (weight.shape != (K,) or weight.dtype not in (dtype, torch.float32) or weight.device != device or
                               not weight.is_contiguous()):
        raise ValueError("rms_norm: weight must be a dense [K] tensor on x's device, of x's dtype or fp32")
    if residual_out is not None and residual is None:
        raise ValueError("rms_norm: residual_out without a residual")
    if out is not None and not store:
        raise ValueError("rms_norm: out with store=False")
    if out is not None:
        _like("out", out, shape, dtype, device)
    if residual_out is not None:
        _like("residual_out", residual_out, shape, dtype, device)
    y = None if not store else x.new_empty(shape) if out is None else out
    if residual is not None:
        _like("residual", residual, shape, dtype, device)
        if residual_out is None:
            residual_out = x.new_empty(shape)
    codes = scales = None
    if quant == "fp8":
        codes, scales = x.new_empty(shape, dtype=torch.float8_e4m3fn), x.new_empty(shape[:-1], dtype=torch.float32)
    elif quant == "mxfp4":
        if K % 32:
            raise ValueError("rms_norm: MXFP4 codes need K to be a multiple of 32")
        codes, scales = x.new_empty((*shape[:-1], K // 2), dtype=torch.uint8), x.new_empty((*shape[:-1], K // 32), dtype=torch.uint8)
    n = _lib.ObRmsNorm(shape[0], H, K, _ROWS[dtype], 0 if weight is None else _WEIGHT[weight.dtype], _QUANT[quant], eps,
                       *_rows(x, dims), None if weight is None else weight.data_ptr(),
                       *(_NO_ROWS if residual is None else _rows(residual, dims)),
                       *(_NO_ROWS if residual_out is None else _rows(residual_out, dims)),
                       *(_NO_ROWS if y is None else _rows(y, dims)),
                       None if codes is None else codes.data_ptr(), None if scales is None else scales.data_ptr())
    _lib.call_on(device, "ob_rms_norm", C.byref(n))
    return NormOut(y, residual_out, codes, scales)
