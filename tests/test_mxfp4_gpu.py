"""MXFP4 quantization and its inverse: bit-exact against the 64-bit oracle (every step is exact arithmetic, so there is no
tolerance) over types, sizes, strides, every rounding border and the ends of the exponent range."""
from __future__ import annotations

import pytest
import torch

from oracle import mxfp4 as omx

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _q(x, **k):
    from onebase_b200.kernels.mxfp4 import quantize
    r = quantize(x, **k)
    torch.cuda.synchronize()
    return r


def _dq(*a, **k):
    from onebase_b200.kernels.mxfp4 import dequantize
    r = dequantize(*a, **k)
    torch.cuda.synchronize()
    return r


def _same(x):
    c, s = _q(x)
    rc, rs = omx.quant(x)
    assert torch.equal(s.cpu(), rs)
    assert torch.equal(c.cpu(), rc)
    return c, s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (5, 96), (1, 4096), (33, 1056), (130, 7392), (2, 3, 160), (64,), (7, 12288)])
def test_random_tensors(shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=g) * torch.exp2(torch.randint(-12, 9, shape, generator=g).float())).to(dtype).cuda()
    c, s = _same(x)
    want = omx.dequant(c, s)
    for out in TYPES:
        v = _dq(c, s, out)
        assert v.shape == x.shape and torch.equal(v.cpu(), want.to(out))


@pytest.mark.parametrize("shape", [(0, 32), (0, 5, 64)])
def test_no_rows(shape):
    c, s = _q(torch.empty(shape, dtype=torch.bfloat16, device="cuda"))
    assert c.shape[-1] == shape[-1] // 2 and _dq(c, s).shape == shape


def test_rounding_borders_and_saturation():
    """Every border of e2m1, the fp32 values next to it on both sides, and everything from 6 to the largest a block can hold."""
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.0, 0.5])
    probes = torch.cat([border, torch.nextafter(border, torch.tensor(100.0)), torch.nextafter(border, torch.tensor(-100.0))])
    probes = torch.cat([probes, -probes])
    for e in (-100, -3, 0, 5, 100):
        rows = torch.zeros(len(probes), 32)
        rows[:, 0] = 7.5                       # the block's largest: exponent 2, scale 2^0
        rows[:, 7] = probes
        rows[:, 31] = -probes
        _same((rows * 2.0 ** e).cuda())


@pytest.mark.parametrize("dtype", TYPES)
def test_ends_of_the_range(dtype):
    fi = torch.finfo(dtype)
    rows = torch.zeros(8, 64, dtype=dtype)
    rows[0, 3] = fi.max
    rows[1, 3] = fi.smallest_normal
    rows[2, 3] = fi.smallest_normal * fi.eps              # the smallest subnormal
    rows[3, :32] = fi.smallest_normal
    rows[4, 40] = -fi.max
    rows[5] = -0.0
    rows[6, 5], rows[6, 6] = fi.max, fi.smallest_normal
    rows[7, :32] = torch.linspace(-1, 1, 32).to(dtype) * fi.smallest_normal * 4
    c, s = _same(rows.cuda())
    want = omx.dequant(c, s)
    assert torch.equal(_dq(c, s, torch.float32).cpu(), want.float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nan_and_infinite_blocks(dtype, bad):
    x = torch.randn(4, 128, generator=torch.Generator().manual_seed(9)).to(dtype)
    clean = x.clone()
    x[1, 40] = bad
    c, s = _same(x.cuda())
    assert int(s[1, 1]) == 255 and int((s == 255).sum()) == 1
    v = _dq(c, s, dtype)
    assert bool(torch.isnan(v[1, 32:64]).all()) and int(torch.isnan(v).sum()) == 32
    rc, rs = omx.quant(clean)
    keep = torch.ones_like(v, dtype=torch.bool)
    keep[1, 32:64] = False
    assert torch.equal(v.cpu()[keep.cpu()], omx.dequant(rc, rs).to(dtype)[keep.cpu()])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 8), (3, 0), (0, 1), (32, 4)])
def test_strided_rows(dtype, pad, offset):
    M, K = 9, 96
    g = torch.Generator().manual_seed(pad)
    buf = torch.randn(M * (K + pad) + offset, generator=g).to(dtype).cuda()
    x = buf[offset:].view(M, K + pad)[:, :K]
    c, s = _same(x)
    keep = buf.clone()
    out = buf[offset:].view(M, K + pad)[:, :K]
    _dq(c, s, out=out)
    assert torch.equal(out.cpu(), omx.dequant(c, s).to(dtype))
    keep[offset:].view(M, K + pad)[:, :K] = out
    assert torch.equal(buf, keep)                          # nothing between the rows was written


def test_transposed_and_broadcast_inputs():
    x = torch.randn(64, 96, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    _same(x.t()[:, :64])                                    # columns of x as rows
    _same(x[:1].expand(5, 96))


def test_given_outputs_and_graph():
    x = torch.randn(17, 2048, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    c, s = torch.full((17, 1024), 7, dtype=torch.uint8, device="cuda"), torch.full((17, 64), 7, dtype=torch.uint8, device="cuda")
    r = _q(x, codes=c, scales=s)
    assert r[0].data_ptr() == c.data_ptr() and torch.equal(c.cpu(), omx.quant(x)[0])
    from onebase_b200.kernels.mxfp4 import dequantize, quantize
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v = dequantize(*quantize(x))
    x.copy_(x.flip(1).contiguous())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(v.cpu(), omx.dequant(*omx.quant(x)).to(torch.bfloat16))


def test_more_than_two_to_the_32_elements():
    M, K = 65537, 65536
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("not enough free device memory")
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    probe = torch.randn(2, K, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    x[0], x[M - 1] = probe[0].cuda(), probe[1].cuda()
    c, s = _q(x)
    rc, rs = omx.quant(probe)
    for at, i in ((0, 0), (M - 1, 1)):
        assert torch.equal(c[at].cpu(), rc[i]) and torch.equal(s[at].cpu(), rs[i])
    assert int(c[1: M - 1].sum(dtype=torch.int64)) == 0
    x.fill_(1.0)
    _dq(c, s, out=x)
    assert torch.equal(x[M - 1].cpu(), omx.dequant(rc[1], rs[1]).to(torch.bfloat16)) and not bool(x[1: M - 1].any())
