"""An MXFP4 base takes the large tiles from 65 tokens: a layer's own workspace has room for them, so that a call runs the same kernels
whether the layer stands alone on its device or beside larger ones, and ob_resolve_tile names what runs."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from helpers import device_meta, make_index
from onebase_b200 import _lib
from onebase_b200.kernels import fp8_lora_vllm
from oracle import configs, mxfp4 as omx, segments as oseg


@pytest.mark.parametrize("max_m,max_l,lc", [(64, 4, 0), (65, 4, 4), (96, 0, 0), (128, 200, 128), (129, 7, 7)])
def test_room_for_the_per_tenant_blocks(max_m, max_l, lc):
    s = _lib.ObWorkspaceShape(max_m, 1024, 1024, 128, 32, 8, max_l)
    off, n = C.c_size_t(), C.c_size_t()
    _lib.call("ob_workspace_region", C.byref(s), _lib.OB_WS["hcat"], C.byref(off), C.byref(n))
    want = 128 * max_m * lc * 2
    assert want <= n.value < want + 1024


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,R,M", [("bf16", 64, 80), ("nvfp4", 32, 65), ("bf16", 128, 96)])
def test_alone_and_beside_a_larger_layer(monkeypatch, fmt, R, M):
    from test_mxfp4_lora_gpu import _case, _ok, _op, check, reference
    monkeypatch.setattr(fp8_lora_vllm, "_SCRATCH", {})                   # a device of this test's own
    d = _case(1024, (520, 256), R, 5, M, seed=M)
    op = _op(d, 96, lora_fmt=fmt)
    assert op.scratch.shape.max_m == 96 and op.resolved_tile(M)["prefill"] == 1
    meta, x = device_meta(make_index(d["ids"], 5, 96), M), d["x"].cuda()
    alone = op(x, meta)
    _ok(op)
    check(alone, reference(op, d, d["x"], d["ids"]))
    rows, _ = oseg.resolve_positions(M, *[t.cpu() for t in meta])
    q, sf = omx.quant(d["x"])
    for tn in (None, 256):                                               # the scales lie as the large tiles read them
        xq, xsf = op.codes(M, tn)
        assert torch.equal(xq.cpu(), q[rows]) and torch.equal(xsf.cpu(), sf[rows])
    larger = _op(_case(2048, (640,), 16, 9, 8), 700)
    assert larger.scratch is op.scratch and op.scratch.shape.max_m == 700
    beside = op(x, meta)
    _ok(op)
    assert torch.equal(alone, beside)
