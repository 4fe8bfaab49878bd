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
