"""Operands written in place and read by the next projection, whose kernels read weights, scales and adapters before their wait on the
launch in front of them: between the two lies a launch without the programmatic attribute (seen in the captured graph's edges), and the call
sees the new values."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from helpers import build_fp8_op, build_nvfp4_op, device_meta, make_index
from oracle import configs
from test_mxfp4_lora_gpu import _case, _ok, _op, check, reference

pytestmark = pytest.mark.gpu


class EdgeData(C.Structure):
    _fields_ = [("from_port", C.c_ubyte), ("to_port", C.c_ubyte), ("type", C.c_ubyte), ("reserved", C.c_ubyte * 5)]


def captured(call):
    """The edges of the graph `call` makes: (from, to) node numbers in the order of the nodes -> 0 (full) or 1 (programmatic)."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    edges_of = C.CDLL("libcuda.so.1").cuGraphGetEdges_v2
    edges_of.argtypes = [C.c_void_p] * 5
    n, raw = C.c_size_t(), C.c_void_p(graph.raw_cuda_graph())
    assert edges_of(raw, None, None, None, C.addressof(n)) == 0
    a, b, data = (C.c_void_p * n.value)(), (C.c_void_p * n.value)(), (EdgeData * n.value)()
    assert edges_of(raw, a, b, data, C.addressof(n)) == 0
    n = n.value
    chain = {x: (y, d.type) for x, y, d in zip(a, b, data)}
    assert len(chain) == n                                    # one chain: no node has two successors
    node = next(iter(set(chain) - {y for y, _ in chain.values()}))
    types = []
    while node in chain:
        node, t = chain[node]
        types.append(t)
    return graph, types


def test_a_weight_quantized_in_place_lies_behind_a_fence():
    from onebase_b200.kernels.mxfp4 import quantize
    M, K, L = 9, 512, 3
    d = _case(K, (256,), 16, L, M)
    op = _op(d, 16)
    meta, x = device_meta(make_index(d["ids"], L, 16), M), d["x"].cuda()
    w = d["w"].to(torch.bfloat16).cuda()
    sf = torch.empty_like(op.w_sf)
    op(x, meta)
    y = torch.empty(M, 256, dtype=torch.bfloat16, device="cuda")

    def update():
        quantize(w, codes=op.w_q, scales=sf)                  # (the packed scales stay: the new weight has the old one's)
        op(x, meta, out=y)

    graph, types = captured(update)
    assert types == [0, 1, 1]                                 # quantizer, fence, K1, K2
    old = op.w_q.clone()
    w.neg_()
    graph.replay()
    _ok(op)
    assert not torch.equal(op.w_q, old) and torch.equal(sf, op.w_sf)
    d["w_mx"] = op.w_q.cpu()
    check(y, reference(op, d, d["x"], d["ids"]))
    # outputs of its own are activations: no fence, and the projection starts beside the quantizer
    _, types = captured(lambda: op(x, meta, out=y, quantized=quantize(x)))
    assert types == [1, 1]


def test_an_adapter_dequantized_in_place_lies_behind_a_fence():
    from onebase_b200.kernels.mxfp4 import dequantize, quantize
    M, K, L = 5, 512, 3
    d = _case(K, (256,), 16, L, M)
    op = _op(d, 16)
    meta, x = device_meta(make_index(d["ids"], L, 16), M), d["x"].cuda()
    codes, scales = quantize(op.a_stacked[0][1, 0])
    op(x, meta)
    _, types = captured(lambda: (dequantize(codes, scales, out=op.a_stacked[0][1, 0]), op(x, meta)))
    assert types == [0, 1, 1]


@pytest.mark.parametrize("base", ["nvfp4", "mxfp4"])
def test_packed_weight_scales(base):
    K, widths = 512, (200, 72)
    if base == "mxfp4":
        from onebase_b200.kernels.mxfp4_lora_vllm import pack_weight_scales
        sf = torch.zeros(272, K // 32, dtype=torch.uint8, device="cuda")
    else:
        from onebase_b200.kernels.nvfp4_lora_vllm import pack_weight_scales
        sf = torch.zeros(272, K // 16, dtype=torch.uint8, device="cuda")
    _, types = captured(lambda: pack_weight_scales(sf, K, widths))
    assert types == [0]                                       # the re-layout, the fence


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "nvfp4"])
def test_an_adapter_slot_refreshed(fmt):
    M, K, L = 7, 256, 3
    d = configs.draw(K, (128,), 16, L, M, seed=3)
    for op in (build_fp8_op(configs.with_fp8_base(d), 16, lora_fp8=fmt == "fp8", lora_fp4=fmt == "nvfp4"),
               build_nvfp4_op(configs.with_nvfp4_base(d), 16, lora_fmt=fmt)):
        meta, x = device_meta(make_index(d["ids"], L, 16), M), d["x"].cuda()
        op(x, meta)

        def refresh():
            op.a_stacked[0][1].mul_(2)
            op.requantize(1)
            op(x, meta)

        _, types = captured(refresh)
        assert types[-3:] == [0, 1, 1]                        # ..., fence, K1, K2
        assert types[:-2] == [0] * (len(types) - 2)
