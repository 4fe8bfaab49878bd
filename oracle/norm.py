"""Oracle (test infrastructure, CPU torch, 64-bit): root-mean-square norm with a residual in front (RMSNorm.forward_native,
vllm/model_executor/layers/layernorm.py, in 64 bits) and the FP8 row scale behind."""
from __future__ import annotations

import torch

FP8_MAX, MIN_SCALE = 448.0, 1.0 / (448.0 * 512.0)


def rms_norm(x, weight, eps, residual=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(s, y) in float64: s = x + residual, y = s / sqrt(mean(s^2) + eps) * weight."""
    s = x.double().cpu() if residual is None else x.double().cpu() + residual.double().cpu()
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, y if weight is None else y * weight.double().cpu()


def fp8_scale(y: torch.Tensor) -> torch.Tensor:
    return (y.abs().amax(-1) / FP8_MAX).clamp(min=MIN_SCALE)
