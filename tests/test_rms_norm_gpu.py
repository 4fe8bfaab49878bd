"""rms_norm against a 64-bit evaluation: types, rows of one element to long ones, head views, strides, in-place use, quantised
outputs, rows of zeros and rows with a NaN.

Tolerances.  u = 2^-24 is half a step of fp32.  The kernel's y carries, relative to the exact one: the sum s (u), two products (2u),
the sum of squares (at most K/16 + 16 additions in a row, half of it under the root), the division, the addition of eps,
the root and its reciprocal (4u) -- below (K/32 + 16) u -- and the store's rounding, eps(T)/2.  A code is off by half a step of its
format relative to its value (e4m3: 2^-4) or half a subnormal step (2^-10 scales), on top of the fp32 error."""
from __future__ import annotations

import pytest
import torch

from oracle import mxfp4 as omx, norm as onorm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _norm(*a, **k):
    from onebase_b200.kernels.rms_norm import rms_norm
    r = rms_norm(*a, **k)
    torch.cuda.synchronize()
    return r


def _inputs(shape, dtype, seed=0, wdtype=None, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * 2).to(dtype)
    x[..., :: max(1, shape[-1] // 3)] *= 8
    r = torch.randn(shape, generator=g).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(shape[-1], generator=g)).to(wdtype or dtype)
    return x, w, r


def fp32_err(K):
    return (K / 32 + 16) * U


def check_y(y, ref, K):
    dt = y.dtype
    fi = torch.finfo(dt)
    sub = fi.smallest_normal * fi.eps / 2
    err = (y.double().cpu() - ref).abs()
    tol = ref.abs() * ((1 + fp32_err(K)) * (1 + fi.eps / 2) - 1) + sub
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp_min(1e-300)).max()):.3f} of the tolerance"


def check_fp8(codes, scales, ref, K):
    rs = onorm.fp8_scale(ref)
    assert bool(((scales.double().cpu() - rs).abs() <= rs * (fp32_err(K) + 2 * U)).all())
    sc = scales.double().cpu().unsqueeze(-1)
    v = codes.cpu().double() * sc
    tol = ref.abs() * (2.0 ** -4 + 2 * fp32_err(K)) + sc * 2.0 ** -10
    assert bool(((v - ref).abs() <= tol).all())


def check_mx(codes, scales, ref, K):
    d = 2 * fp32_err(K)
    got = scales.cpu()
    lo, hi = omx.scale_bytes(ref * (1 - d)), omx.scale_bytes(ref * (1 + d))
    assert bool(((got == lo) | (got == hi)).all())
    # codes: those of ref under the kernel's scale, wherever no rounding border lies within the fp32 error
    c = omx.unpack(codes.cpu())
    same_lo, same_hi = omx.codes_of(ref * (1 - d), got), omx.codes_of(ref * (1 + d), got)
    assert bool(((c == same_lo) | (c == same_hi)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (2, 8), (5, 33), (1, 64), (7, 96), (4, 128), (3, 255), (17, 256), (2, 1000), (9, 1024),
                                 (3, 2048), (2, 2056), (33, 4096), (2, 4100), (3, 7392), (2, 8192), (3, 12288), (1, 16384), (2, 29568), (1, 40000)])
def test_norm_of_rows(M, K, dtype):
    x, w, r = _inputs((M, K), dtype, seed=M + K)
    n = _norm(x.cuda(), w.cuda(), 1e-6, residual=r.cuda(), quant="fp8")
    s, y = onorm.rms_norm(x, w, 1e-6, r)
    assert torch.equal(n.residual.cpu(), (x.float() + r.float()).to(dtype))
    check_y(n.y, y, K)
    check_fp8(n.codes, n.scales, y, K)
    p = _norm(x.cuda(), w.cuda(), 1e-6)
    assert p.residual is None and p.codes is None and p.scales is None
    check_y(p.y, onorm.rms_norm(x, w, 1e-6)[1], K)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", [(1, 32), (5, 64), (3, 128), (9, 288), (2, 1024), (7, 1056), (33, 4096), (2, 7392), (3, 12288), (1, 16416), (1, 40000)])
def test_mxfp4_codes(M, K, dtype):
    x, w, r = _inputs((M, K), dtype, seed=M * K)
    n = _norm(x.cuda(), w.cuda(), 1e-5, residual=r.cuda(), quant="mxfp4")
    _, y = onorm.rms_norm(x, w, 1e-5, r)
    check_y(n.y, y, K)
    check_mx(n.codes, n.scales, y, K)


@pytest.mark.parametrize("wdtype", [torch.float32, None, "none"])
@pytest.mark.parametrize("K", [128, 4096, 77])
def test_weights(K, wdtype):
    x, w, _ = _inputs((6, K), torch.bfloat16, wdtype=torch.float32 if wdtype is torch.float32 else None)
    w = None if wdtype == "none" else w
    n = _norm(x.cuda(), None if w is None else w.cuda(), 1e-6, quant="fp8")
    _, y = onorm.rms_norm(x, w, 1e-6)
    check_y(n.y, y, K)
    check_fp8(n.codes, n.scales, y, K)


@pytest.mark.parametrize("quant", [None, "fp8", "mxfp4"])
@pytest.mark.parametrize("M,H,K,tail", [(5, 3, 64, 0), (4, 8, 128, 2 * 128), (1, 32, 128, 1024), (3, 2, 96, 5), (2, 5, 256, 8), (0, 4, 128, 0)])
def test_heads_of_a_merged_row(M, H, K, tail, quant):
    """[M, H, K] views of rows that go on behind the heads (keys and values), normed into place and out of place."""
    g = torch.Generator().manual_seed(H)
    wide = torch.randn(M, H * K + tail, generator=g).to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(K, generator=g)).to(torch.bfloat16)
    dev = wide.cuda()
    view = dev[:, : H * K].unflatten(1, (H, K))
    _, y = onorm.rms_norm(wide[:, : H * K].unflatten(1, (H, K)), w, 1e-6)
    n = _norm(view, w.cuda(), 1e-6, quant=quant)
    assert n.y.shape == (M, H, K) and torch.equal(dev.cpu(), wide)
    check_y(n.y, y, K)
    if quant == "fp8":
        check_fp8(n.codes, n.scales, y, K)
    elif quant == "mxfp4":
        check_mx(n.codes, n.scales, y, K)
    inplace = _norm(view, w.cuda(), 1e-6, out=view)
    assert inplace.y.data_ptr() == view.data_ptr() and torch.equal(view, n.y)
    assert torch.equal(dev[:, H * K:].cpu(), wide[:, H * K:])             # what lies behind the heads is left as it was


@pytest.mark.parametrize("K,pad,offset", [(64, 8, 0), (64, 3, 0), (4096, 8, 8), (4096, 0, 1), (1000, 24, 0), (12288, 16, 0)])
def test_strides_and_alignment(K, pad, offset):
    M = 5
    g = torch.Generator().manual_seed(K)
    base = torch.randn(3, M * (K + pad) + offset + 8, generator=g).to(torch.bfloat16).cuda()
    x, r, o = (b[offset: offset + M * (K + pad)].view(M, K + pad)[:, :K] for b in base)
    keep = base.clone()
    w = torch.ones(K, dtype=torch.bfloat16, device="cuda")
    _, y = onorm.rms_norm(x, w, 1e-6, r)
    s = (x.float() + r.float()).to(torch.bfloat16)
    n = _norm(x, w, 1e-6, residual=r, out=o, quant="fp8")
    check_y(o, y, K)
    check_fp8(n.codes, n.scales, y, K)
    assert torch.equal(n.residual, s)
    changed = base != keep
    mask = torch.zeros_like(changed)
    mask[2, offset: offset + M * (K + pad)].view(M, K + pad)[:, :K] = True
    assert not bool((changed & ~mask).any())                              # nothing but `out` was written
    # the residual stream updated in place, x overwritten by the norm
    n2 = _norm(x, w, 1e-6, residual=r, residual_out=r, out=x)
    assert torch.equal(r, s) and torch.equal(x, o) and n2.residual.data_ptr() == r.data_ptr()


def test_broadcast_row_and_one_row_many_times():
    x = torch.randn(1, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    n = _norm(x.expand(7, 256), torch.ones(256, dtype=torch.bfloat16, device="cuda"), 1e-6, quant="mxfp4")
    one = _norm(x, torch.ones(256, dtype=torch.bfloat16, device="cuda"), 1e-6, quant="mxfp4")
    assert all(torch.equal(n.y[i], one.y[0]) and torch.equal(n.codes[i], one.codes[0]) for i in range(7))


@pytest.mark.parametrize("K", [96, 4096, 12288, 40000])
def test_zero_rows_nan_rows_and_infinities(K):
    x = torch.randn(5, K, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    x[1] = 0
    x[2, K // 2] = float("nan")
    x[3, K - 1] = float("inf")
    w = torch.ones(K, dtype=torch.bfloat16)
    f = _norm(x.cuda(), w.cuda(), 1e-6, quant="fp8")
    m = _norm(x.cuda(), w.cuda(), 1e-6, quant="mxfp4")
    assert bool((f.y[1] == 0).all()) and float(f.scales[1]) == float(torch.tensor(onorm.MIN_SCALE, dtype=torch.float32)) and bool((f.codes[1].float() == 0).all())
    assert bool((m.scales[1] == 0).all()) and bool(((m.codes[1] & 0x77) == 0).all())
    assert bool(torch.isnan(f.y[2]).all()) and bool(torch.isnan(f.scales[2])) and bool(torch.isnan(f.codes[2].float()).all())
    assert bool((m.scales[2] == 255).all()) and bool((m.codes[2] == 0).all())
    assert bool(torch.isnan(f.y[3, K - 1])) and bool((f.y[3, : K - 1] == 0).all())
    assert bool(torch.isnan(f.scales[3])) and bool(torch.isnan(f.codes[3].float()).all())
    assert int(m.scales[3, -1]) == 255
    _, y = onorm.rms_norm(x, w, 1e-6)
    for i in (0, 4):                                                      # the other rows do not notice
        check_y(f.y[i], y[i], K)
        check_fp8(f.codes[i], f.scales[i], y[i], K)
        check_mx(m.codes[i], m.scales[i], y[i], K)


def test_store_off_gives_the_same_codes():
    x, w, r = _inputs((9, 2048), torch.bfloat16)
    a = _norm(x.cuda(), w.cuda(), 1e-6, residual=r.cuda(), quant="fp8")
    b = _norm(x.cuda(), w.cuda(), 1e-6, residual=r.cuda(), quant="fp8", store=False)
    assert b.y is None and torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.residual, b.residual)


def test_runs_alike_and_in_a_graph_on_another_stream():
    x, w, r = (t.cuda() for t in _inputs((37, 4096), torch.bfloat16))
    a = _norm(x, w, 1e-6, residual=r, quant="fp8")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    from onebase_b200.kernels.rms_norm import rms_norm
    with torch.cuda.stream(side):
        b = rms_norm(x, w, 1e-6, residual=r, quant="fp8")
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = rms_norm(x, w, 1e-6, residual=r, quant="fp8")
    x2 = x.flip(0).contiguous()
    x.copy_(x2)
    graph.replay()
    d = _norm(x2, w, 1e-6, residual=r, quant="fp8")
    for i in range(4):
        assert torch.equal(a[i].view(torch.uint8), b[i].view(torch.uint8))
        assert torch.equal(c[i].view(torch.uint8), d[i].view(torch.uint8))


def test_offsets_beyond_32_bits():
    """Rows 2^21 elements apart, 1100 of them: the last ones begin behind 2^31 elements."""
    M, K, ld = 1100, 64, 1 << 21
    if torch.cuda.mem_get_info()[0] < 3 * M * ld * 2:
        pytest.skip("not enough free device memory")
    base = torch.zeros(M * ld, dtype=torch.bfloat16, device="cuda")
    x = base.view(M, ld)[:, :K]
    x.copy_(torch.randn(M, K, generator=torch.Generator().manual_seed(5)))
    w = torch.ones(K, dtype=torch.bfloat16, device="cuda")
    dense = x.contiguous()
    _norm(x, w, 1e-6, out=x)
    assert torch.equal(x, _norm(dense, w, 1e-6).y)
