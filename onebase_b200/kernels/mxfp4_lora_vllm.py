"""Fused MXFP4 (W4A4) base + multi-tenant LoRA for one vLLM LoRA layer, on B200 through libonebase_b200.so.

The third base format beside FP8 and NVFP4, with the same call, batches, adapters and fused neighbours: W as e2m1 codes packed two
per byte along K ([N, K/2] uint8, element 2i in the low nibble) with one power-of-two scale per 32 elements ([N, K/32] uint8,
exponent + 127) -- OCP microscaling, what mxfp4.quantize makes of a weight --, x quantized to the same format on the fly, or
given in codes (`quantized=`); y = alpha * sum(v(x) v(w)) + LoRA.  No global scale and no calibration: an activation's scale
follows its own block.  The reference has no counterpart (its 4-bit base is NVFP4, lowbit_lora/kernels/nvfp4_lora_vllm.py:437-630).
"""
from __future__ import annotations

import ctypes as C

import torch

from onebase_b200 import _lib
from onebase_b200.kernels import mxfp4
from onebase_b200.kernels.adapter_store import AdapterStore
from onebase_b200.kernels.fp8_lora_vllm import Scratch, VllmFusedFP8LoRA, fill_adapter_pointers, shared_scratch


def pack_weight_scales(w_sf: torch.Tensor, K: int, widths) -> torch.Tensor:
    """Linear [N, K/32] scale bytes -> the per-(tile, K slot) atom order K2 copies to TMEM (one kernel launch)."""
    if not w_sf.is_cuda or not w_sf.is_contiguous() or w_sf.element_size() != 1 or tuple(w_sf.shape) != (sum(widths), K // 32):
        raise ValueError("pack_weight_scales: w_sf must be a dense one-byte [sum(widths), K/32] CUDA tensor")
    wa = (C.c_int32 * len(widths))(*widths)
    n = C.c_size_t()
    _lib.call("ob_mxfp4_packed_scale_bytes", K, len(widths), wa, C.byref(n))
    out = torch.empty(n.value, dtype=torch.uint8, device=w_sf.device)
    _lib.call_on(w_sf.device, "ob_mxfp4_pack_scales", w_sf.data_ptr(), K, len(widths), wa, out.data_ptr(), n.value)
    return out


class VllmFusedMXFP4LoRA(VllmFusedFP8LoRA):
    """w_q [N, K/2] uint8 (packed e2m1), w_sf [N, K/32] uint8 (exponent + 127), K a multiple of 32; a_stacked / b_stacked vLLM's
    per-slice bf16 adapter buffers, kept as `lora_fmt` ("bf16", "fp8" or "nvfp4"); alpha scales the base product."""

    _K1, _K2, _CHAIN, _FMT = "ob_k1_mxfp4", "ob_k2_mxfp4", "ob_chain_mxfp4", "mxfp4"

    def __init__(self, w_q, w_sf, a_stacked, b_stacked, max_m, *, alpha: float = 1.0, split_k=None, lora_fmt="bf16"):
        if w_q.device.type != "cuda":
            raise RuntimeError("onebase_b200 runs on CUDA devices only (there is no CPU path)")
        self.w_q, self.w_sf = w_q, w_sf
        self.N, self.K = w_q.shape[0], 2 * w_q.shape[1]
        self.S = len(a_stacked)
        self.L, _, self.R, k_a = a_stacked[0].shape
        if w_q.dtype != torch.uint8 or not w_q.is_contiguous() or w_sf.dtype != torch.uint8 or tuple(w_sf.shape) != (self.N, self.K // 32):
            raise ValueError("VllmFusedMXFP4LoRA: w_q must be dense uint8 [N, K/2], w_sf uint8 [N, K/32]")
        assert k_a == self.K and all(t.dtype == torch.bfloat16 and t.is_contiguous() for t in (*a_stacked, *b_stacked))
        if any(t.device != w_q.device for t in (w_sf, *a_stacked, *b_stacked)):
            raise ValueError("VllmFusedMXFP4LoRA: weight, scales and adapters must be on one device")
        widths = [t.shape[2] for t in b_stacked]
        assert sum(widths) == self.N and self.S <= 4
        ends = [sum(widths[:i + 1]) for i in range(self.S)]
        self.end0 = ends[0] if self.S >= 2 else self.N
        self.end1 = ends[1] if self.S >= 3 else self.N
        self.end2 = ends[2] if self.S >= 4 else self.N
        self.widths = widths
        self.a_stacked, self.b_stacked = a_stacked, b_stacked
        self.max_m = int(max_m)
        self.split_k = split_k
        self.lora_fmt = lora_fmt
        self.lora_fp8, self.lora_fp4 = lora_fmt == "fp8", lora_fmt == "nvfp4"
        self.device = w_q.device
        self.store = AdapterStore(a_stacked, b_stacked, lora_fmt)
        self.alpha = torch.full((1,), float(alpha), dtype=torch.float32, device=self.device)
        self.w_sf_packed = pack_weight_scales(w_sf.contiguous(), self.K, widths)
        self.scratch = shared_scratch(self.device)
        self.scratch.ensure(self.max_m, self.K, self.N, self.S * self.R, Scratch.MAX_SPLIT2, self.L)
        self.dispatch = {}
        self.wait_ms = 2000
        d = _lib.ObLayerDesc()
        d.base_fmt = _lib.OB_BASE_MXFP4
        d.N, d.K, d.S, d.L, d.R, d.max_m = self.N, self.K, self.S, self.L, self.R, self.max_m
        for s in range(self.S):
            d.widths[s] = widths[s]
        fill_adapter_pointers(d, self.store)
        d.w_q, d.w_sf, d.alpha = w_q.data_ptr(), self.w_sf_packed.data_ptr(), self.alpha.data_ptr()
        self._desc = d
        h = C.c_void_p()
        with torch.cuda.device(self.device):
            _lib.call("ob_layer_create", C.byref(d), C.byref(h))
        self._h = h

    @classmethod
    def from_weight(cls, weight: torch.Tensor, a_stacked, b_stacked, max_m, **kw) -> "VllmFusedMXFP4LoRA":
        """The op over a bf16, fp16 or fp32 weight [N, K], quantized here (mxfp4.quantize)."""
        return cls(*mxfp4.quantize(weight), a_stacked, b_stacked, max_m, **kw)

    def _codes_ok(self, codes, scales, M: int) -> bool:
        return (codes.dtype == torch.uint8 and tuple(codes.shape) == (M, self.K // 2) and scales.dtype == torch.uint8 and
                tuple(scales.shape) == (M, self.K // 32))

    def codes(self, M: int, tn: int | None = None):
        """The last call's activation codes and scale bytes in POSITION order: (packed [M, K/2] uint8, [M, K/32] uint8, read back
        out of the scale-factor atoms)."""
        K = self.K
        xq = self.scratch.region("xq", M * (K // 2)).view(M, K // 2)
        if tn is None:   # the token tile the library's own rule gave the last call; 256 under the large-tile prefill GEMM
            rt = self.resolved_tile(M)
            tn = 256 if rt["prefill"] == 1 else rt["tn"]
        nblk = 2 if tn > 128 else 1
        kslots = (K + 255) // 256
        m_tiles = (M + tn - 1) // tn
        raw = self.scratch.region("xsf", m_tiles * kslots * nblk * 1024).view(m_tiles, kslots, nblk, 2, 32, 4, 4)
        # [mt, kb, blk, atom, r32, r4, j] -> [mt, blk, r4, r32, kb, atom, j] = [positions, scale columns]
        lin = raw.permute(0, 2, 5, 4, 1, 3, 6).reshape(m_tiles, nblk * 128, kslots * 8)[:, :tn].reshape(m_tiles * tn, kslots * 8)
        return xq, lin[:M, : K // 32].contiguous()
