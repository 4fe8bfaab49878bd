"""Oracle (test infrastructure, CPU torch, 64-bit): MXFP4 quantization, its inverse, and a projection on an MXFP4 base.

The format is OCP microscaling's: blocks of 32 elements share the scale 2^(floor(log2 max|v|) - 2), stored as exponent + 127 (at
least 0; 255 where the block holds an infinity or a NaN), an element is the e2m1 value next to v / scale, ties to even,
saturating at 6.  Packing as the NVFP4 side: element 2i in the low nibble.
"""
from __future__ import annotations

import torch

from oracle.fp8 import lora_term
from oracle.nvfp4 import E2M1_VALUES

BLOCK = 32


def scale_bytes(v: torch.Tensor) -> torch.Tensor:
    """v float64 [..., K] -> uint8 [..., K/32]."""
    top = v.unflatten(-1, (v.shape[-1] // BLOCK, BLOCK)).abs().amax(-1)                 # (amax keeps a NaN)
    exponent = torch.frexp(torch.where(torch.isfinite(top), top, torch.ones_like(top))).exponent - 1
    byte = (exponent - 2 + 127).clamp(min=0)
    byte = torch.where(top == 0, torch.zeros_like(byte), byte)
    return torch.where(torch.isfinite(top), byte, torch.full_like(byte, 255)).to(torch.uint8)


def scale_values(byte: torch.Tensor) -> torch.Tensor:
    return torch.where(byte == 255, torch.full((), float("nan"), dtype=torch.float64), torch.exp2(byte.double() - 127.0))


def codes_of(v: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """v float64 [..., K], scale bytes [..., K/32] -> unpacked codes int64 [..., K]; codes of a NaN block are 0.  The sign bit is the
    value's own, a zero's included."""
    q = v.unflatten(-1, (v.shape[-1] // BLOCK, BLOCK)) / scale_values(byte).unsqueeze(-1)
    grid = torch.tensor(E2M1_VALUES, dtype=torch.float64)
    a = q.abs().clamp(max=6.0)
    dist = (a.unsqueeze(-1) - grid).abs()
    best = dist.amin(-1, keepdim=True)
    # nearest value; of two equally near ones the even code
    order = torch.arange(8) % 2
    mag = torch.where(dist == best, order, 9).argmin(-1)
    code = mag + 8 * torch.signbit(q).long()
    return torch.where(torch.isnan(q), torch.zeros_like(code), code).reshape(v.shape)


def pack(codes: torch.Tensor) -> torch.Tensor:
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def unpack(packed: torch.Tensor) -> torch.Tensor:
    p = packed.long()
    return torch.stack((p & 15, p >> 4), -1).flatten(-2)


def quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] of any float type -> (packed codes, scale bytes)."""
    v = x.double().cpu()
    byte = scale_bytes(v)
    return pack(codes_of(v, byte)), byte


def dequant(packed: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """float64 values."""
    c = unpack(packed.cpu())
    v = torch.tensor(E2M1_VALUES, dtype=torch.float64)[c & 7] * torch.where(c >= 8, -1.0, 1.0).double()
    return (v.unflatten(-1, (v.shape[-1] // BLOCK, BLOCK)) * scale_values(byte.cpu()).unsqueeze(-1)).flatten(-2)


def fused_projection(x, token_lora, w_q, w_sf, a, b, widths, alpha: float = 1.0, xq=None, xsf=None) -> torch.Tensor:
    """alpha dequant(x_q) dequant(W)^T + LoRA on x itself; fp32 [M, N]."""
    if xq is None:
        xq, xsf = quant(x)
    base = alpha * (dequant(xq, xsf) @ dequant(w_q, w_sf).t())
    return base.float() + lora_term(x, token_lora, a, b, widths, 1.0)
