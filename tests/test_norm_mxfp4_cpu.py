"""Refusals of the norm and of the MXFP4 quantizer, without a GPU: the C entry points turn bad arguments down before any launch,
the Python calls raise.  The oracle's own rounding is held to a table."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from onebase_b200 import _lib
from oracle import mxfp4 as omx

FAKE = 0x10000                                            # never dereferenced on the host


def norm_status(**over):
    n = _lib.ObRmsNorm()
    n.M, n.H, n.K, n.dtype, n.quant, n.eps = 4, 1, 64, _lib.OB_DTYPE_BF16, _lib.OB_QUANT_FP8, 1e-6
    n.x = n.weight = FAKE
    n.x_ld = n.y_ld = n.residual_out_ld = n.residual_ld = 64
    n.y = n.codes = n.scales = 2 * FAKE
    for k, v in over.items():
        setattr(n, k, v)
    return _lib.lib().ob_rms_norm(C.byref(n), None)


@pytest.mark.parametrize("over,status", [
    ({"M": -1}, -2), ({"H": 0}, -2), ({"K": 0}, -2), ({"M": 1 << 20, "H": 1 << 12}, -2),
    ({"dtype": _lib.OB_DTYPE_F32}, -6), ({"dtype": 9}, -6), ({"weight_dtype": _lib.OB_DTYPE_F16}, -6), ({"quant": 3}, -6),
    ({"quant": _lib.OB_QUANT_MXFP4, "K": 48}, -2), ({"eps": -1.0}, -2), ({"eps": float("nan")}, -2),
    ({"x": None}, -1), ({"codes": None}, -1), ({"scales": None}, -1), ({"y": None, "quant": _lib.OB_QUANT_NONE}, -1),
    ({"x_ld": -64}, -2), ({"residual": FAKE, "residual_ld": -1}, -2),
    ({"y_ld": 32}, -2), ({"y_ld": 0}, -2), ({"H": 2, "y_ld": 64, "y_hd": 32}, -2), ({"H": 2, "y_ld": 64, "y_hd": 64}, -2),
    ({"residual": FAKE, "residual_out": 3 * FAKE, "residual_out_ld": 63}, -2),
    ({"residual": FAKE, "residual_out": 2 * FAKE}, -2),                       # two outputs in one place
    ({"x": FAKE + 1}, -3), ({"y": FAKE + 1}, -3), ({"codes": FAKE + 4}, -3), ({"scales": FAKE + 2}, -3),
    ({"weight_dtype": _lib.OB_DTYPE_F32, "weight": FAKE + 2}, -3),
])
def test_norm_refuses(over, status):
    assert norm_status(**over) == status


def test_norm_of_no_tokens_launches_nothing():
    assert norm_status(M=0) == 0 and norm_status(M=0, x=None, codes=None) == 0
    assert _lib.lib().ob_rms_norm(None, None) == -1


@pytest.mark.parametrize("args,status", [
    ((FAKE, 7, 4, 64, 64, FAKE, FAKE), -6), ((FAKE, 0, -1, 64, 64, FAKE, FAKE), -2), ((FAKE, 0, 4, 48, 64, FAKE, FAKE), -2),
    ((FAKE, 0, 4, 0, 64, FAKE, FAKE), -2), ((FAKE, 0, 4, 64, -1, FAKE, FAKE), -2), ((None, 0, 4, 64, 64, FAKE, FAKE), -1),
    ((FAKE, 0, 4, 64, 64, None, FAKE), -1), ((FAKE, 0, 4, 64, 64, FAKE, None), -1), ((FAKE, 0, 4, 64, 64, FAKE + 2, FAKE), -3),
    ((FAKE + 2, 1, 4, 64, 64, FAKE, FAKE), -3), ((None, 0, 0, 64, 64, None, None), 0), ((FAKE, 0, 1 << 60, 64, 64, FAKE, FAKE), -2),
])
def test_quantize_refuses(args, status):
    x, dt, rows, K, ld, codes, scales = args
    assert _lib.lib().ob_mxfp4_quantize(x, dt, rows, K, ld, codes, scales, None) == status
    if x is not None or rows == 0:
        assert _lib.lib().ob_mxfp4_dequantize(codes, scales, dt, rows, K, x, ld, None) == status


def test_dequantize_refuses_rows_on_top_of_each_other():
    assert _lib.lib().ob_mxfp4_dequantize(FAKE, FAKE, 0, 2, 64, FAKE, 32, None) == -2


def test_no_cpu_path():
    from onebase_b200.kernels.mxfp4 import dequantize, quantize
    from onebase_b200.kernels.rms_norm import rms_norm
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: rms_norm(x, None), lambda: quantize(x),
                 lambda: dequantize(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8))):
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            call()


def test_oracle_rounds_by_the_table():
    v = torch.zeros(2, 32, dtype=torch.float64)
    v[0, :12] = torch.tensor([7.5, 0.25, 0.2500001, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.0001, -0.75, -6.5])
    byte = omx.scale_bytes(v)
    assert byte.tolist() == [[127], [0]]
    assert omx.codes_of(v, byte)[0, :12].tolist() == [7, 0, 1, 2, 2, 4, 4, 6, 6, 7, 10, 15]
    assert omx.scale_bytes(torch.full((1, 32), float("inf"))).item() == 255


def test_mxfp4_base_shards():
    """MXFP4 base under tensor parallelism (shard arithmetic, the oracle standing in for the kernels): column shards concatenate to the
    unsharded result, row shards -- whose activation codes equal the unsharded ones block for block -- sum to it."""
    from onebase_b200 import tp
    from oracle import configs, fp8 as ofp8
    world = 2
    d = configs.with_mxfp4_base(configs.draw(256, (128, 64), 16, 4, 11, seed=13, w_std=0.05, b_std=0.05))
    A, B = ofp8.stack_slices(d["a_stacked"], d["b_stacked"])
    full = omx.fused_projection(d["x"], d["ids"], d["w_mx"], d["w_mx_sf"], A, B, d["widths"])
    parts, total = [], torch.zeros_like(full)
    for rank in range(world):
        q_r, sf_r, a_r, b_r = tp.shard_column_mxfp4(d["w_mx"], d["w_mx_sf"], d["a_stacked"], d["b_stacked"], world, rank)
        assert q_r.shape == (96, 128) and sf_r.shape == (96, 8)
        parts.append(omx.fused_projection(d["x"], d["ids"], q_r, sf_r, *ofp8.stack_slices(a_r, b_r), [t.shape[2] for t in b_r]))
        q_r, sf_r, a_r, b_r = tp.shard_row_mxfp4(d["w_mx"], d["w_mx_sf"], d["a_stacked"], d["b_stacked"], world, rank)
        assert q_r.shape == (192, 64) and sf_r.shape == (192, 4) and a_r[0].shape[-1] == 128
        x_r = tp.shard_input_row(d["x"], world, rank)
        assert torch.equal(omx.quant(x_r)[1], omx.quant(d["x"])[1][:, rank * 4:(rank + 1) * 4])
        total += omx.fused_projection(x_r, d["ids"], q_r, sf_r, *ofp8.stack_slices(a_r, b_r), d["widths"])
    cols, off = [], 0
    for w in d["widths"]:
        cols.append(torch.cat([p[:, off // world: (off + w) // world] for p in parts], 1))
        off += w
    assert torch.equal(torch.cat(cols, 1), full)
    # a rank rounds its partial h to bf16: at most half a step of it, against the term's largest value
    assert float((total - full).abs().max() / full.abs().max()) <= 2 * 2.0 ** -8
    with pytest.raises(AssertionError):
        tp.shard_row_mxfp4(d["w_mx"][:, :24], d["w_mx_sf"][:, :1], d["a_stacked"], d["b_stacked"], world, 0)


@pytest.mark.parametrize("over,status", [
    ({"w_sf": None}, -1), ({"alpha": None}, -1), ({"K": 272}, -2), ({"w_q": 0x10004}, -3), ({"w_sf": 0x10004}, -3), ({"base_fmt": 3}, -6),
])
def test_mxfp4_layer_refuses(over, status):
    d = _lib.ObLayerDesc()
    d.base_fmt, d.lora_fmt = _lib.OB_BASE_MXFP4, 0
    d.N, d.K, d.S, d.L, d.R, d.max_m = 256, 256, 2, 4, 16, 8
    d.widths[0], d.widths[1] = 128, 128
    d.w_q = d.w_sf = d.alpha = FAKE
    for s in range(2):
        d.a[s], d.b[s] = FAKE, FAKE
    for k, v in over.items():
        setattr(d, k, v)
    h = C.c_void_p()
    assert _lib.lib().ob_layer_create(C.byref(d), C.byref(h)) == status and not h.value


def test_mxfp4_packed_scale_sizes_and_refusals():
    lib, n = _lib.lib(), C.c_size_t()
    w = (C.c_int32 * 2)(200, 72)
    assert lib.ob_mxfp4_packed_scale_bytes(288, 2, w, C.byref(n)) == 0 and n.value == 3 * 2 * 1024
    assert lib.ob_mxfp4_packed_scale_bytes(272, 2, w, C.byref(n)) == -2 and lib.ob_mxfp4_packed_scale_bytes(288, 5, w, C.byref(n)) == -2
    assert lib.ob_mxfp4_packed_scale_bytes(288, 2, w, None) == -1 and lib.ob_mxfp4_packed_scale_bytes(288, 2, None, C.byref(n)) == -1
    assert lib.ob_mxfp4_pack_scales(FAKE, 288, 2, w, FAKE, 6143, None) == -4
    assert lib.ob_mxfp4_pack_scales(None, 288, 2, w, FAKE, 6144, None) == -1
    assert lib.ob_k1_mxfp4(None, None, None, None, None, None) == -1
    assert lib.ob_k2_mxfp4(None, None, None, None, None, 0, None) == -1
    assert lib.ob_chain_mxfp4(None, None, None, None, None, None) == -1
