"""The norm's FP8 codes where y / scale is a tie of e4m3: rows of small integers, whose sum of squares is exact in fp32 in any order, so that
every step behind it -- division, root, reciprocal, products, quotient -- is one IEEE operation that numpy repeats.  Codes and scales have to
be those of the rounded quotient, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top,K", [(224, 64), (224, 256), (112, 1000), (56, 4096), (28, 4096), (100, 256), (28, 8192), (28, 16384), (224, 63),
                                   (112, 257), (56, 1001), (28, 4095), (28, 9001), (28, 20001)])
def test_codes_of_ties(top, K, dtype):
    from onebase_b200.kernels.rms_norm import rms_norm
    M = 150
    g = np.random.default_rng(top + K)
    s = g.integers(-top, top + 1, (M, K)).astype(F)
    s[:, 0], s[:, 1] = top, -0.0
    total = (s.astype(np.float64) ** 2).sum(-1)
    assert total.max() < 2 ** 24
    y = s * (F(1) / np.sqrt(total.astype(F) / F(K) + F(1e-6)))[:, None]
    scale = np.abs(y).max(-1) / F(448)
    q = torch.from_numpy(np.clip(y / scale[:, None], -448, 448))
    want = q.to(torch.float8_e4m3fn)
    assert q.dtype == torch.float32
    n = rms_norm(torch.from_numpy(s).to(dtype).cuda(), None, 1e-6, quant="fp8")
    assert torch.equal(n.scales.cpu(), torch.from_numpy(scale))
    assert torch.equal(n.codes.cpu().view(torch.uint8), want.view(torch.uint8))
