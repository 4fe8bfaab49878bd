"""Projections on an MXFP4 base through the C ABI: activation codes and scale bytes bit-exact against the oracle, outputs against a
64-bit evaluation, over decode and prefill kernels, every adapter storage, ragged sizes, fused neighbours, given codes.

Tolerance of an output element: half a step of bf16 for its store (2^-8 |y|; twice with a residual), half a step of bf16 for every h
(2^-8 |h| |B|, also where B itself is a stored code times its scale), and fp32 sums of K and of R terms whose products are
exact or rounded once (K 2^-24 |x| |W|, (K + R) 2^-24 |x| |A| |B|)."""
from __future__ import annotations

import pytest
import torch

from helpers import device_meta, make_index, stored_adapters
from oracle import configs, mxfp4 as omx, neighbours as onb, segments as oseg

pytestmark = pytest.mark.gpu


def _case(K, widths, R, L, M, seed=0):
    d = configs.draw(K, widths, R, L, M, seed=seed, ids_low=-1, w_std=0.05, b_std=0.05)
    d["x"][:, :3] *= 8
    return configs.with_mxfp4_base(d)


def _op(d, max_m, **kw):
    from onebase_b200.kernels.mxfp4_lora_vllm import VllmFusedMXFP4LoRA
    return VllmFusedMXFP4LoRA(d["w_mx"].cuda(), d["w_mx_sf"].cuda(), tuple(t.cuda() for t in d["a_stacked"]),
                              tuple(t.cuda() for t in d["b_stacked"]), max_m, **kw)


def _ok(op):
    torch.cuda.synchronize()
    st = op.scratch.status()
    assert st[0] == 0, f"device status {st[:8]}"


def reference(op, d, x, ids, alpha=1.0, residual=None, codes=None):
    """(y, tolerance) in float64 on the GPU (plain matrix products)."""
    packed, byte = codes or omx.quant(x)
    A, B = (t.double().cuda() for t in stored_adapters(op, op.lora_fmt))
    xq, w, xd = (t.double().cuda() for t in (omx.dequant(packed, byte), omx.dequant(d["w_mx"], d["w_mx_sf"]), x))
    y = alpha * (xq @ w.t())
    K, R = x.shape[1], op.R
    tol = abs(alpha) * K * 2.0 ** -24 * (xq.abs() @ w.abs().t())
    for l in torch.unique(ids).tolist():
        if l < 0:
            continue
        rows = torch.nonzero(ids == l).flatten().cuda()
        off = 0
        for s, n in enumerate(d["widths"]):
            a, b = A[l, s * R:(s + 1) * R], B[l, off: off + n]
            h, ha = xd[rows] @ a.t(), xd[rows].abs() @ a.abs().t()
            y[rows, off: off + n] += h @ b.t()
            tol[rows, off: off + n] += 2.0 ** -8 * (h.abs() @ b.abs().t()) * (2 if op.lora_fmt != "bf16" else 1) + (K + R) * 2.0 ** -24 * (ha @ b.abs().t())
            off += n
    if residual is not None:
        tol += 2.0 ** -8 * y.abs()
        y = y + residual.double().cuda()
    return y, tol + 2.0 ** -8 * (y.abs() + tol) + 2.0 ** -120


def check(y, ref_tol, what=""):
    ref, tol = ref_tol
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float(((y.double() - ref).abs() / tol).max()):.2f} of the tolerance"


def _kind_ids(kind, L, M, max_m, idx, g):
    idx.prepare(torch.randint(0, L, (max_m,), generator=g, dtype=torch.int32))      # what an earlier batch left behind
    if kind == "none":
        ids = torch.full((M,), -1, dtype=torch.int32)
    elif kind == "single":
        ids = torch.full((M,), L - 1, dtype=torch.int32)
    elif kind == "all":
        ids = torch.arange(M, dtype=torch.int32) % L
    else:
        ids = torch.randint(-1, L, (M,), generator=g, dtype=torch.int32)
    if kind == "padded":
        ids[0] = 0
        idx.srt[M - 5:M] = 10 ** 6
        idx.tok[M - 5:M] = L - 1
        idx.prepare(ids[: M - 5])
        ids[M - 5:] = -1
    else:
        idx.prepare(ids)
    return ids


@pytest.mark.parametrize("K,widths,R,L,M,kind", [
    (32, (16,), 16, 1, 1, "single"),
    (256, (128, 128), 16, 4, 16, "mixed"),
    (64, (32, 16, 16), 16, 4, 21, "mixed"),
    (96, (64,), 32, 3, 5, "mixed"),
    (512, (256,), 64, 8, 13, "none"),
    (1024, (384, 128), 64, 6, 40, "single"),
    (128, (64,), 128, 2, 24, "padded"),
    (2048, (256, 128, 128), 32, 32, 32, "all"),
    (4096, (512,), 64, 6, 100, "mixed"),
    (7392, (264,), 16, 4, 7, "mixed"),
    (4096, (136, 72, 40, 8), 256, 2, 3, "mixed"),
    (1056, (1, 3), 16, 2, 9, "mixed"),
])
def test_decode_and_small_tiles(K, widths, R, L, M, kind):
    d = _case(K, widths, R, L, M, seed=K + M)
    op = _op(d, 128)
    g = torch.Generator().manual_seed(7)
    idx = oseg.SegmentIndex(L, 128)
    ids = _kind_ids(kind, L, M, 128, idx, g)
    meta_cpu, meta = idx.args(M), device_meta(idx, M)
    x = d["x"].cuda()
    y = op(x, meta)
    _ok(op)
    rows, _ = oseg.resolve_positions(M, *meta_cpu)
    q_ref, sf_ref = omx.quant(d["x"])
    xq, xsf = op.codes(M)
    assert torch.equal(xq.cpu(), q_ref[rows]) and torch.equal(xsf.cpu(), sf_ref[rows])
    check(y, reference(op, d, d["x"], ids))
    from onebase_b200.kernels.mxfp4 import quantize
    for kw in ({"pdl": False}, {"cfg": {"fused": 1}}, {"cfg": {"stream": 1}}, {"quantized": quantize(x)}):
        assert torch.equal(y, op(x, meta, **kw)), kw
        _ok(op)


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("K,M,tn,split2,stages", [
    (4096, 30, 32, 1, 2), (4096, 30, 32, 4, 0), (4096, 30, 32, 8, 3), (4096, 9, 16, 7, 2), (4096, 60, 64, 2, 0), (4096, 120, 128, 1, 0),
    (4096, 300, 64, 1, 0), (4096, 300, 32, 1, 4), (992, 300, 0, 0, 0), (4064, 129, 0, 0, 0), (4096, 16, 16, 1, 12)])
def test_token_tiles_splits_and_rings(K, M, tn, split2, stages, fmt):
    d = _case(K, (264, 120), 64, 5, M, seed=M + K)
    op = _op(d, 320, lora_fmt=fmt)
    idx = make_index(d["ids"], 5, 320)
    cfg = {k: v for k, v in (("tn", tn), ("split2", split2), ("stages", stages)) if v}
    y = op(d["x"].cuda(), device_meta(idx, M), cfg=cfg)
    _ok(op)
    check(y, reference(op, d, d["x"], d["ids"]))
    y2 = op(d["x"].cuda(), device_meta(idx, M), cfg=cfg, pdl=False)
    _ok(op)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("fmt,R", [("bf16", 64), ("bf16", 16), ("bf16", 256), ("fp8", 128), ("nvfp4", 64)])
@pytest.mark.parametrize("K,widths,M,L", [(4096, (520, 128, 136), 33, 7), (8192, (1024, 128, 128), 64, 32), (12288, (640,), 47, 3), (512, (2048, 2052), 64, 5), (4096, (8192, 8192), 40, 4), (4064, (24,), 63, 64)])
def test_one_tile_of_up_to_64_tokens(K, widths, M, L, fmt, R):
    d = _case(K, widths, R, L, M, seed=M + K)
    op = _op(d, 64, lora_fmt=fmt)
    idx = make_index(d["ids"], L, 64)
    y = op(d["x"].cuda(), device_meta(idx, M))
    _ok(op)
    check(y, reference(op, d, d["x"], d["ids"]))
    for kw in ({"cfg": {"prefill": 1}}, {"cfg": {"prefill": 2}}):
        y2 = op(d["x"].cuda(), device_meta(idx, M), **kw)
        _ok(op)
        check(y2, reference(op, d, d["x"], d["ids"]), kw)
    y3 = op(d["x"].cuda(), device_meta(idx, M), pdl=False)
    _ok(op)
    assert torch.equal(y, y3)


@pytest.mark.parametrize("fmt,R", [("bf16", 64), ("bf16", 16), ("fp8", 64), ("nvfp4", 32), ("bf16", 256), ("nvfp4", 128)])
@pytest.mark.parametrize("K,widths,M,L", [(256, (256,), 129, 4), (1024, (264, 128), 65, 6), (2048, (640,), 128, 3), (1024, (520, 104), 200, 32), (2048, (384, 8, 128), 777, 7), (512, (4096,), 3000, 5), (1056, (264,), 300, 3), (32, (128,), 140, 2), (7392, (136, 256), 260, 4)])
def test_large_prefill_tiles(K, widths, M, L, fmt, R):
    """The CTA-pair kernel: ragged tokens and slices, several tiles per pair, every storage."""
    d = _case(K, widths, R, L, M, seed=K + M + R)
    d["ids"] = configs.zipf_request_ids(M, L, seed=M)
    op = _op(d, 3000, lora_fmt=fmt)
    meta = device_meta(make_index(d["ids"], L, M), M)
    assert op.resolved_tile(M, {"prefill": 1})["prefill"] == 1
    y = op(d["x"].cuda(), meta, cfg={"prefill": 1})
    _ok(op)
    xq, xsf = op.codes(M, tn=256)
    rows, _ = oseg.resolve_positions(M, *[t.cpu() for t in meta])
    q_ref, sf_ref = omx.quant(d["x"])
    assert torch.equal(xq.cpu(), q_ref[rows]) and torch.equal(xsf.cpu(), sf_ref[rows])
    check(y, reference(op, d, d["x"], d["ids"]))
    from onebase_b200.kernels.mxfp4 import quantize
    assert torch.equal(y, op(d["x"].cuda(), meta, cfg={"prefill": 1}, quantized=quantize(d["x"].cuda())))
    assert torch.equal(y, op(d["x"].cuda(), meta, cfg={"prefill": 1}))
    _ok(op)


@pytest.mark.parametrize("M", [1, 9, 31, 100, 257, 600])
@pytest.mark.parametrize("silu,residual", [(True, False), (False, True), (True, True)])
def test_fused_neighbours(M, silu, residual):
    K, widths, L = 1536, (320,), 4
    d = _case(K, widths, 16, L, M, seed=M)
    op = _op(d, 640)
    g = torch.Generator().manual_seed(M)
    meta = device_meta(make_index(d["ids"], L, 640), M)
    x_in = torch.randn(M, 2 * K, generator=g).to(torch.bfloat16) if silu else d["x"]
    x = onb.silu_mul(x_in) if silu else x_in
    res = torch.randn(M, 320, generator=g).to(torch.bfloat16) if residual else None
    y = op(x_in.cuda(), meta, silu_mul=silu, residual=None if res is None else res.cuda())
    _ok(op)
    if silu:   # silu's exponential may round a bf16 of the input the other way: the codes the kernel made are what is held to the sum
        rows, _ = oseg.resolve_positions(M, *[t.cpu() for t in meta])
        xq, xsf = (t.cpu() for t in op.codes(M))
        back = torch.empty_like(rows)
        back[rows] = torch.arange(M)
        codes = (xq[back], xsf[back])
        ref_codes = omx.quant(x)
        assert float((codes[0] != ref_codes[0]).float().mean()) < 1e-2
    else:
        codes = None
    check(y, reference(op, d, x, d["ids"], residual=res, codes=codes))
    if res is not None:                                    # in place on the stream
        yr = res.cuda()
        assert torch.equal(op(x_in.cuda(), meta, silu_mul=silu, residual=yr, out=yr), y)


def test_silu_of_infinite_and_far_gates():
    """The prefill quantizer's cheaper quotient against the decode batch's IEEE division: gates where it would leave its range."""
    K, M = 1024, 300
    d = _case(K, (128,), 16, 2, M, seed=5)
    op = _op(d, 320)
    idx = make_index(torch.full((M,), -1), 2, 320)
    x = torch.zeros(M, 2 * K)
    gates = torch.tensor([float("inf"), float("-inf"), float("nan"), -86.5, -87.5, -88.0, -88.5, -89.0, -120.0, -3e38, 3e38, -0.0, 1e-40, -1e-40])
    ups = torch.tensor([1.0, -2.0, 3e38, 2.0 ** 120])
    x[:, K:] = 1.0
    for r in range(16):                              # a block of 32 per (gate, up): the gate in its first element
        for b in range(32):
            k = r * 32 + b
            x[r, b * 32], x[r, K + b * 32] = gates[k % len(gates)], ups[(k // len(gates)) % len(ups)]
    x = x.to(torch.bfloat16).cuda()
    op(x[:16], device_meta(make_index(torch.full((16,), -1), 2, 320), 16), silu_mul=True)
    _ok(op)
    few = [t[:16].clone() for t in op.codes(16)]
    op(x, device_meta(idx, M), silu_mul=True)
    _ok(op)
    many = [t[:16] for t in op.codes(M)]
    assert torch.equal(few[1], many[1]) and torch.equal(few[0], many[0])
    assert int((few[1] == 255).sum()) >= 16 * 32 // len(gates) * 2     # (at least the gates of -inf and NaN)


@pytest.mark.parametrize("M", [3, 70, 300])
def test_alpha_scales_and_far_apart_blocks(M):
    """Weight scales over many powers of two, blocks of zeros, an alpha that is no power of two."""
    K, widths, L = 512, (128, 64), 3
    d = _case(K, widths, 16, L, M, seed=M)
    g = torch.Generator().manual_seed(3)
    d["w_mx_sf"] = torch.randint(100, 150, d["w_mx_sf"].shape, generator=g, dtype=torch.uint8)
    d["w_mx_sf"][:, 3] = 0
    d["w_mx"][5] = 0
    op = _op(d, 320, alpha=0.7)
    meta = device_meta(make_index(d["ids"], L, 320), M)
    y = op(d["x"].cuda(), meta)
    _ok(op)
    check(y, reference(op, d, d["x"], d["ids"], alpha=float(torch.tensor(0.7))))


@pytest.mark.parametrize("M,K", [(4, 256), (40, 1056), (300, 512)])
def test_nan_and_infinite_tokens_keep_to_themselves(M, K):
    d = _case(K, (136,), 16, 3, M, seed=M)
    d["ids"][:] = torch.arange(M, dtype=torch.int32) % 3
    op = _op(d, 320)
    meta = device_meta(make_index(d["ids"], 3, 320), M)
    clean = op(d["x"].cuda(), meta).clone()
    x = d["x"].clone()
    x[1, 7], x[2, K - 1] = float("nan"), float("inf")
    y = op(x.cuda(), meta)
    _ok(op)
    assert bool(torch.isnan(y[1:3]).all())
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])


def test_strided_inputs_and_outputs_and_rows_behind_the_batch():
    M, K, L = 37, 1024, 4
    d = _case(K, (200, 56), 32, L, M)
    op = _op(d, 64)
    meta = device_meta(make_index(d["ids"], L, 64), M)
    want = op(d["x"].cuda(), meta)
    wide = torch.zeros(M, K + 24, dtype=torch.bfloat16, device="cuda")
    wide[:, :K] = d["x"].cuda()
    out = torch.full((M + 4, 256 + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    y = op(wide[:, :K], meta, out=out[:M, :256])
    _ok(op)
    assert torch.equal(y, want) and bool((out[M:] == 7).all()) and bool((out[:, 256:] == 7).all())


def test_captured_and_replayed_with_other_inputs():
    M, K, L = 24, 2048, 6
    d = _case(K, (256, 128), 64, L, M)
    op = _op(d, 32)
    meta = device_meta(make_index(d["ids"], L, 32), M)
    x = d["x"].cuda()
    from onebase_b200.kernels.mxfp4 import quantize
    op(x, meta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = op(x, meta)
        z = op(x, meta, quantized=quantize(x))
    x.copy_(x.flip(0).contiguous())
    for _ in range(3):
        graph.replay()
    _ok(op)
    assert torch.equal(y, z)
    check(y, reference(op, d, x.cpu(), d["ids"]))


@pytest.mark.parametrize("base", ["fp8", "mxfp4"])
@pytest.mark.parametrize("M", [1, 16, 77, 300])
def test_norm_hands_its_codes_to_the_projection(M, base):
    """The run of the operators together: residual and norm, codes handed on, projection; two layers' worth, in one graph and
    eagerly, against the 64-bit evaluation of each step on the step's own inputs."""
    from helpers import build_fp8_op
    from onebase_b200.kernels.rms_norm import rms_norm
    from oracle import fp8 as ofp8, norm as onorm
    K, L = 1024, 5
    d = _case(K, (K,), 32, L, M, seed=M)
    configs.with_fp8_base(d)
    op = _op(d, 320) if base == "mxfp4" else build_fp8_op(d, 320)
    meta = device_meta(make_index(d["ids"], L, 320), M)
    g = torch.Generator().manual_seed(M)
    stream = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    w = (1 + 0.2 * torch.randn(K, generator=g)).to(torch.bfloat16).cuda()
    x = d["x"].cuda()

    def step():
        n1 = rms_norm(x, w, 1e-6, residual=stream, quant=base)
        y1 = op(n1.y, meta, quantized=(n1.codes, n1.scales))
        n2 = rms_norm(y1, w, 1e-6, residual=n1.residual, quant=base)
        return n1, y1, n2, op(n2.y, meta, quantized=(n2.codes, n2.scales))

    eager = step()
    _ok(op)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    _ok(op)
    for a, b in zip(eager, captured):
        for s, t in zip(a if isinstance(a, tuple) else [a], b if isinstance(b, tuple) else [b]):
            assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))
    n1, y1, n2, y2 = eager
    for n, y in ((n1, y1), (n2, y2)):
        if base == "mxfp4":
            check(y, reference(op, d, n.y.cpu(), d["ids"], codes=(n.codes.cpu(), n.scales.cpu())))
        else:
            A, B = ofp8.stack_slices(d["a_stacked"], d["b_stacked"])
            ref = ofp8.fused_projection(n.y.cpu(), d["ids"], d["w_q"], d["s_w"], A, B, d["widths"], xq=n.codes.cpu(), sx=n.scales.cpu())
            assert float((y.float().cpu() - ref).abs().max()) <= 2e-2 * float(ref.abs().max())
    s1, _ = onorm.rms_norm(x, w, 1e-6, stream)
    assert torch.equal(n1.residual.cpu().double(), s1.float().to(torch.bfloat16).double())


@pytest.mark.parametrize("K,M", [(512, 5), (4096, 32), (4096, 100), (12288, 17), (512, 300), (4096, 1100)])
def test_fp8_base_takes_given_codes(K, M):
    """The FP8 projection with its own quantizer's codes given: the same bits."""
    from helpers import build_fp8_op
    from oracle import fp8 as ofp8
    d = configs.with_fp8_base(configs.draw(K, (256, 64), 32, 4, M, seed=K + M))
    op = build_fp8_op(d, 1280)
    meta = device_meta(make_index(d["ids"], 4, 1280), M)
    x = d["x"].cuda()
    codes, scales = ofp8.quant_per_token(d["x"])
    y = op(x, meta)
    z = op(x, meta, quantized=(codes.cuda(), scales.cuda()))
    _ok(op)
    assert torch.equal(y, z)


def test_refusals():
    from helpers import build_fp8_op, build_nvfp4_op
    from onebase_b200._lib import ObError
    from onebase_b200.kernels.mxfp4 import quantize
    from onebase_b200.kernels.mxfp4_lora_vllm import VllmFusedMXFP4LoRA
    d = _case(256, (128,), 16, 2, 8)
    op = _op(d, 8)
    meta = device_meta(make_index(d["ids"], 2, 8), 8)
    x = d["x"].cuda()
    c, s = quantize(x)
    for bad in ((c[:4], s[:4]), (c, s[:, :4]), (c.float(), s), (c, s.float()), (c.cpu(), s), (c.t().contiguous().t(), s)):
        with pytest.raises(ValueError):
            op(x, meta, quantized=bad)
    with pytest.raises(ValueError):
        op(torch.cat([x, x], 1), meta, silu_mul=True, quantized=(c, s))
    with pytest.raises(ValueError):
        VllmFusedMXFP4LoRA(op.w_q, op.w_sf[:, :4], op.a_stacked, op.b_stacked, 8)
    with pytest.raises(ValueError):
        VllmFusedMXFP4LoRA(op.w_q, op.w_sf.cpu(), op.a_stacked, op.b_stacked, 8)
    nv = build_nvfp4_op(configs.with_nvfp4_base(d), 8)
    with pytest.raises(ValueError):
        nv(x, meta, quantized=(c, s))
    fp8 = build_fp8_op(configs.with_fp8_base(d), 8)
    with pytest.raises(ValueError):
        fp8(x, meta, quantized=(c, s))
    with pytest.raises(ObError):
        op(torch.cat([x, x]), device_meta(make_index(torch.zeros(16, dtype=torch.int32), 2, 16), 16))     # more tokens than max_m
    y = op(x, meta)
    _ok(op)
    check(y, reference(op, d, d["x"], d["ids"]))


def test_from_weight_and_scale_packing():
    from onebase_b200.kernels.mxfp4_lora_vllm import VllmFusedMXFP4LoRA, pack_weight_scales
    d = _case(288, (200, 72), 16, 2, 5)
    w = d["w"].to(torch.bfloat16).cuda()
    op = VllmFusedMXFP4LoRA.from_weight(w, tuple(t.cuda() for t in d["a_stacked"]), tuple(t.cuda() for t in d["b_stacked"]), 8)
    assert torch.equal(op.w_q.cpu(), d["w_mx"]) and torch.equal(op.w_sf.cpu(), d["w_mx_sf"])
    K, widths = 1312, (200, 72)
    sf = torch.randint(1, 255, (272, K // 32), dtype=torch.uint8)
    v = pack_weight_scales(sf.cuda(), K, widths).cpu().view(3, 6, 2, 32, 4, 4)      # [tile, K slot, atom, r32, r4, j]
    row0 = tile = 0
    for wd in widths:
        for tl in range((wd + 127) // 128):
            blk = v[tile].permute(3, 2, 0, 1, 4).reshape(128, 48)
            n = min(128, wd - tl * 128)
            assert torch.equal(blk[:n, : K // 32], sf[row0 + tl * 128: row0 + tl * 128 + n])
            assert int(blk[n:].sum()) == 0 and int(blk[:, K // 32:].sum()) == 0
            tile += 1
        row0 += wd


@pytest.mark.parametrize("split2,me", [(1, 0), (3, 1)])
def test_fused_allreduce_with_a_hand_played_peer(split2, me):
    """ob_chain_allreduce on this base: the peer's staged partial and announcements are in the buffers before the launch, so nothing
    waits for another kernel; y is the rank-ordered fp32 sum of both partials, rounded once."""
    from test_fused_allreduce_gpu import HandComm
    K, widths, L, M = 1024, (384, 128), 4, 19
    d = _case(K, widths, 32, L, M, seed=21)
    op = _op(d, 32)
    meta, x = device_meta(make_index(d["ids"], L, 32), M), d["x"].cuda()
    cfg = {"split2": split2}
    part = op(x, meta, cfg=cfg).clone()
    torch.cuda.synchronize()
    hc = HandComm(slot_bytes=32 * 512 * 2, me=me)
    g = torch.Generator(device="cuda").manual_seed(7)
    for epoch in (1, 2):
        theirs = (torch.randn(M, 512, device="cuda", generator=g) * 0.5).to(torch.bfloat16)
        hc.staged(1 - me, epoch & 1, M, 512).copy_(theirs)
        hc.tile_flags(me)[1 - me, :4] = epoch
        y = torch.full_like(part, float("nan"))

        class Peer:
            comm = hc.comm
        op(x, meta, out=y, cfg=cfg, allreduce=Peer)
        _ok(op)
        parts = [part, theirs] if me == 0 else [theirs, part]
        assert torch.equal(y, (parts[0].float() + parts[1].float()).to(torch.bfloat16))
        assert torch.equal(hc.staged(me, epoch & 1, M, 512), part) and bool((hc.tile_flags(1 - me)[me, :4] == epoch).all())


def test_two_layers_share_a_workspace_in_two_graphs():
    """Two captured graphs of two layers over one workspace, replayed in turn on one stream."""
    d1, d2 = _case(1024, (256,), 16, 3, 20, seed=1), _case(2048, (128, 64), 32, 5, 90, seed=2)
    op1, op2 = _op(d1, 32), _op(d2, 128)
    m1, m2 = device_meta(make_index(d1["ids"], 3, 32), 20), device_meta(make_index(d2["ids"], 5, 128), 90)
    x1, x2 = d1["x"].cuda(), d2["x"].cuda()
    w1, w2 = op1(x1, m1).clone(), op2(x2, m2).clone()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for op, x, m in ((op1, x1, m1), (op2, x2, m2)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(op(x, m))
        graphs.append(gr)
    for i in (0, 1, 1, 0, 1, 0):
        graphs[i].replay()
    _ok(op1)
    assert torch.equal(outs[0], w1) and torch.equal(outs[1], w2)
    check(w2, reference(op2, d2, d2["x"], d2["ids"]))


def test_calls_from_another_current_device(monkeypatch):
    """Each entry makes its tensors' device current for the launch and leaves the caller's as it was."""
    from onebase_b200.kernels.mxfp4 import dequantize, quantize
    from onebase_b200.kernels.rms_norm import rms_norm
    d = _case(256, (128,), 16, 2, 5)
    op = _op(d, 64)
    x, meta = d["x"].cuda(), device_meta(make_index(d["ids"], 2, 64), 5)
    want = op(x, meta), rms_norm(x, None).y, quantize(x)[0], dequantize(*quantize(x))
    state = {"current": 1, "made": []}

    class Guard:
        def __init__(self, device):
            self.index = device if isinstance(device, int) else torch.device(device).index

        def __enter__(self):
            self.before, state["current"] = state["current"], self.index
            state["made"].append(self.index)

        def __exit__(self, *exc):
            state["current"] = self.before

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    codes, scales = quantize(x)
    got = op(x, meta), rms_norm(x, None).y, codes, dequantize(codes, scales)
    monkeypatch.undo()
    _ok(op)
    assert state["made"] == [0] * 4 and state["current"] == 1
    assert all(torch.equal(a, b) for a, b in zip(want, got))
