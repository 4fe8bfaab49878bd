"""SiLU * mul in front of an MXFP4 base's quantizer, held to the definition: every bf16 gate through the prefill quantizer (whose quotient
is an approximate reciprocal with one correction) and through the decode form (IEEE division), and the codes AND scale bytes of random
batches at every size of batch.

The kernels' silu, fp32: expf within 2 ulp (2^-22 relative), the sum and the quotient half a step each -- 2^-22 + 2^-23 relative, half a
subnormal step at most below the normal range -- and then the two bf16 roundings of the activation's definition.  So the input lies between
what the definition gives at both ends of that interval, and its codes between theirs."""
from __future__ import annotations

import pytest
import torch

from helpers import build_fp8_op, device_meta, make_index
from oracle import configs, mxfp4 as omx, segments as oseg
from test_mxfp4_lora_gpu import _case, _ok, _op

pytestmark = pytest.mark.gpu
REL, ABS = 2.0 ** -22 + 2.0 ** -23, 2.0 ** -149


def ends(gate, up):
    """The smallest and the largest bf16 input the definition allows (float64), gates from -87 on."""
    g = gate.double()
    s = g * torch.sigmoid(g)
    room = s.abs() * REL + ABS
    a, b = ((t.to(torch.bfloat16).double() * up.double()).to(torch.bfloat16).double() for t in (s - room, s + room))
    return torch.minimum(a, b), torch.maximum(a, b)


def same_bits(a, b):
    """Equal bit for bit, NaN for NaN."""
    na, nb = torch.isnan(a), torch.isnan(b)
    return torch.equal(na, nb) and torch.equal(a.view(torch.int16)[~na], b.view(torch.int16)[~nb])


@pytest.mark.parametrize("ups", ["one", "random"])
def test_every_gate(ups):
    K = M = 256
    d = _case(K, (128,), 16, 2, M)
    none = torch.full((M,), -1, dtype=torch.int32)
    meta = device_meta(make_index(none, 2, M), M)
    gate = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(M, K)
    up = torch.ones(M, K) if ups == "one" else torch.randn(M, K, generator=torch.Generator().manual_seed(2)) * 3
    up = up.to(torch.bfloat16)
    x = torch.cat([gate, up], 1).cuda()
    op, fp8 = _op(d, M), build_fp8_op(configs.with_fp8_base(d), M)
    inputs = []
    for o in (op, fp8):                                       # the sorted copy of the input, as the adapters see it
        assert o.resolved_tile(M, {"prefill": 1})["prefill"] == 1
        o(x, meta, silu_mul=True, cfg={"prefill": 1})
        _ok(o)
        inputs.append(o.scratch.region("xs", 2 * M * K).view(torch.bfloat16).view(M, K).cpu())
        if o is op:
            codes = [t.cpu() for t in op.codes(M, 256)]
    quick, plain = inputs
    assert same_bits(quick, plain)                            # the FP8 base's quantizer divides
    lo, hi = ends(gate, up)
    near = gate.double() >= -87
    near &= torch.isfinite(gate.double())
    v = quick.double()
    assert bool(((v >= lo) & (v <= hi))[near].all())
    byte = omx.scale_bytes(v)
    assert torch.equal(codes[1], byte) and torch.equal(codes[0], omx.quant(quick)[0])
    few = device_meta(make_index(none[:32], 2, M), 32)
    for r in range(0, M, 32):                                 # the decode form
        op(x[r: r + 32], few, silu_mul=True)
        _ok(op)
        c, s = (t.cpu() for t in op.codes(32))
        assert torch.equal(c, codes[0][r: r + 32]) and torch.equal(s, codes[1][r: r + 32])


@pytest.mark.parametrize("K,M", [(1536, m) for m in (1, 2, 9, 31, 48, 100, 257, 600)] + [(12288, m) for m in (1, 32, 64, 200)])
def test_codes_and_scales(K, M):
    L = 4
    d = _case(K, (320,), 16, L, M, seed=M)
    op = _op(d, 640)
    meta = device_meta(make_index(d["ids"], L, 640), M)
    x = torch.randn(M, 2 * K, generator=torch.Generator().manual_seed(M + K)).to(torch.bfloat16)
    op(x.cuda(), meta, silu_mul=True)
    _ok(op)
    rows, _ = oseg.resolve_positions(M, *[t.cpu() for t in meta])
    codes, byte = (t.cpu() for t in op.codes(M))
    lo, hi = (t[rows] for t in ends(x[:, :K], x[:, K:]))
    small, large = torch.minimum(lo.abs(), hi.abs()), torch.maximum(lo.abs(), hi.abs())
    b = byte.int()
    assert bool(((b >= omx.scale_bytes(small).int()) & (b <= omx.scale_bytes(large).int())).all())
    c = omx.unpack(codes)
    assert bool(((c == omx.codes_of(lo, byte)) | (c == omx.codes_of(hi, byte))).all())
