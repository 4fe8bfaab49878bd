"""The CTA-pair GEMM over an FP4 base where a tile has several times as many expand steps as the ring has slots, few k-blocks, and a pair
walks more than one tile: the block scales' producer and the scale copiers pass the steps by."""
from __future__ import annotations

import pytest
import torch

from helpers import build_nvfp4_op, device_meta, make_index, max_err_ratio, oracle_y_nvfp4, stored_adapters
from oracle import configs, nvfp4 as on4
from test_mxfp4_lora_gpu import _op, check, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("base", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("K,N,R,L,M", [(256, 12288, 128, 60, 700), (1536, 10240, 64, 100, 600)])
def test_many_expand_steps(base, fmt, K, N, R, L, M):
    d = configs.draw(K, (N,), R, L, M, seed=K + M, w_std=0.05, b_std=0.05)
    d["ids"] = torch.arange(M, dtype=torch.int32) % L
    meta, x = device_meta(make_index(d["ids"], L, M), M), d["x"].cuda()
    if base == "mxfp4":
        op = _op(configs.with_mxfp4_base(d), M, lora_fmt=fmt)
    else:
        op = build_nvfp4_op(configs.with_nvfp4_base(d), M, lora_fmt=fmt)
    cfg = {"prefill": 1}
    assert op.resolved_tile(M, cfg)["prefill"] == 1
    y = op(x, meta, cfg=cfg)
    again = op(x, meta, cfg=cfg, out=torch.full_like(y, 7.0))
    torch.cuda.synchronize()
    assert op.scratch.status()[0] == 0, op.scratch.status()[:8]
    assert torch.equal(y, again)
    if base == "mxfp4":
        check(y, reference(op, d, d["x"], d["ids"]))
    elif fmt == "bf16":
        assert max_err_ratio(y, oracle_y_nvfp4(d, d["x"], d["ids"])) <= 2e-2
    else:
        A, B = stored_adapters(op, fmt)
        assert max_err_ratio(y, on4.fused_projection(d["x"], d["ids"], d["w_q4"], d["w_sf"], d["w_global"], d["x_global"], A, B, [N])) <= 2e-2
