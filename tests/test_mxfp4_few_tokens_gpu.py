"""One and two tokens on an MXFP4 base, the form of a single user's decode: against the 64-bit evaluation of test_mxfp4_lora_gpu, over
ragged sizes, ranks, storages, tenants, fused neighbours and what an earlier batch or a padded one leaves in the index."""
from __future__ import annotations

import pytest
import torch

from helpers import device_meta, make_index
from oracle import configs, mxfp4 as omx, neighbours as onb
from test_mxfp4_lora_gpu import _case, _ok, _op, check, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ids", [[0], [-1], [2], [1, 1], [2, 0], [-1, 1], [0, -1], [-1, -1]])
@pytest.mark.parametrize("K,widths", [(32, (5,)), (1024, (16,)), (1056, (1, 3)), (4096, (264, 120, 7)), (7392, (130,)), (12288, (64,))])
def test_tenants_and_ragged_sizes(K, widths, ids):
    M = len(ids)
    d = _case(K, widths, 32, 3, M, seed=K)
    ids = torch.tensor(ids, dtype=torch.int32)
    op = _op(d, 16)
    meta = device_meta(make_index(ids, 3, 16), M)
    x = d["x"].cuda()
    out = torch.full((M + 1, sum(widths) + 3), 5.0, dtype=torch.bfloat16, device="cuda")
    y = op(x, meta, out=out[:M, : sum(widths)])
    _ok(op)
    check(y, reference(op, d, d["x"], ids))
    assert bool((out[M:] == 5).all()) and bool((out[:, sum(widths):] == 5).all())
    for kw in ({"pdl": False}, {}):
        assert torch.equal(y, op(x, meta, **kw))


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("R", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("M", [1, 2])
def test_storages_and_ranks(M, R, fmt):
    d = _case(2048, (96, 40), R, 4, M, seed=R + M)
    d["ids"] = torch.tensor([3, 1][:M], dtype=torch.int32)
    op = _op(d, 8, lora_fmt=fmt, alpha=1.5)
    y = op(d["x"].cuda(), device_meta(make_index(d["ids"], 4, 8), M))
    _ok(op)
    check(y, reference(op, d, d["x"], d["ids"], alpha=1.5))


@pytest.mark.parametrize("M", [1, 2])
@pytest.mark.parametrize("silu,residual", [(True, False), (False, True), (True, True)])
def test_neighbours_and_given_codes(M, silu, residual):
    from onebase_b200.kernels.mxfp4 import quantize
    K = 1536
    d = _case(K, (200,), 16, 2, M, seed=M)
    d["ids"] = torch.tensor([1, 0][:M], dtype=torch.int32)
    op = _op(d, 8)
    meta = device_meta(make_index(d["ids"], 2, 8), M)
    g = torch.Generator().manual_seed(M)
    x_in = torch.randn(M, 2 * K, generator=g).to(torch.bfloat16) if silu else d["x"]
    x = onb.silu_mul(x_in) if silu else x_in
    res = torch.randn(M, 200, generator=g).to(torch.bfloat16) if residual else None
    y = op(x_in.cuda(), meta, silu_mul=silu, residual=None if res is None else res.cuda())
    _ok(op)
    order = meta[1].cpu().long() if bool((d["ids"] >= 0).any()) else torch.arange(M)
    xq, xsf = (t.cpu() for t in op.codes(M))
    back = torch.empty_like(order)
    back[order] = torch.arange(M)
    codes = (xq[back], xsf[back])
    if not silu:
        assert torch.equal(codes[0], omx.quant(x)[0]) and torch.equal(codes[1], omx.quant(x)[1])
        assert torch.equal(y, op(x_in.cuda(), meta, quantized=quantize(x_in.cuda()), residual=None if res is None else res.cuda()))
    check(y, reference(op, d, x, d["ids"], residual=res, codes=codes))
    if res is not None:
        yr = res.cuda()
        assert torch.equal(op(x_in.cuda(), meta, silu_mul=silu, residual=yr, out=yr), y)


def test_nan_token_and_extreme_scales():
    K = 512
    d = _case(K, (64,), 16, 2, 2)
    d["ids"] = torch.tensor([0, 1], dtype=torch.int32)
    d["w_mx_sf"][:, 5] = 0
    d["w_mx_sf"][7] = 160
    op = _op(d, 8)
    meta = device_meta(make_index(d["ids"], 2, 8), 2)
    y = op(d["x"].cuda(), meta).clone()
    _ok(op)
    check(y, reference(op, d, d["x"], d["ids"]))
    x = d["x"].clone()
    x[1, 3] = float("nan")
    z = op(x.cuda(), meta)
    assert bool(torch.isnan(z[1]).all()) and torch.equal(z[0], y[0])
    d["w_mx_sf"][9, 2] = 255                                  # a NaN block of the weight: its row's outputs alone
    n = _op(d, 8)(d["x"].cuda(), meta)
    assert bool(torch.isnan(n[:, 9]).all()) and torch.equal(n[:, :9], y[:, :9]) and torch.equal(n[:, 10:], y[:, 10:])


def test_long_rows():
    K = 51200
    d = _case(K, (24,), 16, 2, 2)
    op = _op(d, 2)
    y = op(d["x"].cuda(), device_meta(make_index(d["ids"], 2, 2), 2))
    _ok(op)
    check(y, reference(op, d, d["x"], d["ids"]))


def test_stale_and_padded_metadata():
    """No-adapter batch behind an adapter batch, and a padded position whose index points anywhere."""
    d = _case(256, (40,), 16, 3, 2)
    op = _op(d, 8)
    idx = make_index(torch.tensor([2, 1], dtype=torch.int32), 3, 8)
    idx.prepare(torch.tensor([-1, -1], dtype=torch.int32))
    y = op(d["x"].cuda(), device_meta(idx, 2))
    _ok(op)
    check(y, reference(op, d, d["x"], torch.tensor([-1, -1])))
    idx.prepare(torch.tensor([1], dtype=torch.int32))
    idx.srt[1], idx.tok[1] = 10 ** 6, 2
    y = op(d["x"].cuda(), device_meta(idx, 2))
    _ok(op)
    check(y, reference(op, d, d["x"], torch.tensor([1, -1])))
