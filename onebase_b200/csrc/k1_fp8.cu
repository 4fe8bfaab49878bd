// K1: activation quantization -- per-token dynamic e4m3 for an FP8 base, e2m1 codes with one ue4m3 scale per 16
// elements against a static global scale for an NVFP4 base, or with one power-of-two scale per 32 for an MXFP4 base; or codes that
// the caller brings -- fused in one launch with every tenant's LoRA shrink
// h = x A^T.
//
// One launch, two kinds of CTA (256 threads each):
//   * CTAs [0, M): quantize one tile POSITION each.  Position p stands for row `position_row(p)` of x: the adapter-sorted
//     order whenever the batch has an adapter, so that K2 can fetch contiguous rows by TMA.  amax over the row in fp32,
//     s_x = max(amax / 448, 1/(448*512)) and code = e4m3_rn(clamp(x / s_x)) with IEEE divisions and ONE rounding step:
//     the rule of lowbit_lora/kernels/fp8_lora_vllm.py:47-71 (vLLM's dynamic per-token quantization), bit for bit.
//   * the remaining CTAs: 8 independent warps each; a warp owns (block of 1 or 4 sorted positions, slice, 8 rank rows,
//     K split) and streams that [8, K/split] block of the positions' adapter A from HBM with 16-byte loads, multiplying it
//     into up to 4 tokens at a time (their x rows come from L2; tokens of one tenant handled by different warps re-read
//     A through L2, not HBM).  The 32 lane-partial sums per warp (8 rank rows x 4 tokens) are
//     reduced with a transposing butterfly -- 31 shuffles for 32 sums, lane i ends up with sum i -- and written as
//     split-K partials hp[split][slice][position][rank] (fp32), which K2 adds in split order (deterministic).
//     Computes what lowbit_lora/kernels/fp8_lora_vllm.py:72-120 computes per adapter segment.
// The kernel starts with griddepcontrol.launch_dependents so that a dependent K2 may begin streaming W at once, and it
// may itself be launched as a programmatic dependent of the preceding kernel: it reads the segment index and requests
// its first block of A before griddepcontrol.wait, and touches x and the scratch only after it.
#include <atomic>

#include "k1_device.cuh"

namespace ob {

constexpr int kK1Threads = 256;

template <int NT, int BASE, int XOP, bool COPY = false>
__device__ __forceinline__ void position_codes(const K1Params& p, int pos, int row, int tid) {
    if constexpr (XOP == OB_X_QUANTIZED) take_row_codes<NT, BASE, COPY>(p, pos, row, tid);
    else if constexpr (BASE == OB_BASE_MXFP4) quantize_row_mxfp4<NT, XOP, COPY>(p, pos, row, tid);
    else if constexpr (BASE == OB_BASE_NVFP4) quantize_row_nvfp4<NT, XOP, COPY>(p, pos, row, tid);
    else quantize_row<NT, 0, XOP, COPY>(p, pos, row, tid);
}

// One instantiation per (adapter storage, base format): each launch carries only the code of its own case.
// LOOPED: the one-CTA-per-SM form that runs beside the persistent GEMM; a function of its own, because the shared-memory
// carve-out it needs (see launch_k1_impl) is a per-function attribute and costs the other form its L1 cache.
// XOP: the projection's input is formed from x on the fly (OB_X_SILU_MUL), or its codes are given (OB_X_QUANTIZED); plain launches run
// an instantiation without either.
template <int LORA_FMT, int BASE, bool LOOPED, int XOP>
__global__ void __launch_bounds__(kK1Threads, XOP == OB_X_SILU_MUL ? 2 : 0) k1_kernel(const K1Params p) {
    griddep_launch_dependents();
    OB_TRACE1(0)
    if ((int)blockIdx.x < p.n_quant_ctas) {
        const int row = row_of_position(p, blockIdx.x, threadIdx.x & 31);
        griddep_wait();                               // x comes from the preceding kernel; the scratch may still be read by it
        position_codes<kK1Threads, BASE, XOP>(p, blockIdx.x, row, threadIdx.x);
        if (p.xs != nullptr) {                        // the tensor-core shrink reads x in position order by TMA
            const __nv_bfloat16* xr = p.x + (int64_t)row * p.ldx;
            uint4* xo = reinterpret_cast<uint4*>(p.xs + (size_t)blockIdx.x * (size_t)p.K);
            for (int i = threadIdx.x; i < (p.K >> 3); i += kK1Threads) xo[i] = x_load8<XOP>(p, xr, i * 8);
        }
        if (p.xq_ready != nullptr) {          // chain: tell K2 that this position's codes and scale are in memory
            __syncthreads();
            if (threadIdx.x == 0) red_release_add(p.xq_ready, 1);
        }
        OB_TRACE1(3)
        if (!LOOPED) return;
    }
    const int lane = threadIdx.x & 31;
    if (LOOPED) {
        // One CTA per SM at most (so that a dependent GEMM's CTAs fit beside this kernel's and stream weights while it
        // runs): every warp of the grid walks the shrink units with the grid's stride; the quantizing CTAs join after
        // their position.
        const long long total = (long long)p.n_pblocks * p.units_per_block;
        const long long stride = (long long)gridDim.x * (kK1Threads / 32);
        for (long long w = (long long)blockIdx.x * (kK1Threads / 32) + (threadIdx.x >> 5); w < total; w += stride)
            shrink_unit<LORA_FMT, XOP>(p, (int)(w / p.units_per_block), (int)(w % p.units_per_block), lane);
        OB_TRACE1(3)
        return;
    }
    const int w = ((int)blockIdx.x - p.n_quant_ctas) * (kK1Threads / 32) + (threadIdx.x >> 5);
    const int pb = w / p.units_per_block;
    if (pb >= p.n_pblocks) return;
    shrink_unit<LORA_FMT, XOP>(p, pb, w % p.units_per_block, lane);
    OB_TRACE1(3)
}

// Quantization alone, for batches whose shrink runs on the tensor cores: without the shrink's registers four of these
// CTAs share an SM instead of two, which is what a launch of thousands of one-row CTAs needs.
template <int BASE, int XOP>
__global__ void __launch_bounds__(kK1Threads, BASE == OB_BASE_MXFP4 ? 8 : 4) k1_quant_kernel(const K1Params p) {
    griddep_launch_dependents();
    const int row = row_of_position(p, blockIdx.x, threadIdx.x & 31);
    griddep_wait();
    position_codes<kK1Threads, BASE, XOP, true>(p, blockIdx.x, row, threadIdx.x);
}

// The FP8 base's form of it with the row in registers (NV vectors per thread of NT threads): one read of x serves the amax, the
// codes and the sorted copy.  MIN_CTAS per SM bounds the registers: the launch is bound by how many rows an SM has in flight
// and, with the input transform, by its instructions.
template <int NT, int NV, int XOP, int MIN_CTAS>
__global__ void __launch_bounds__(NT, MIN_CTAS) k1_quant_regs_kernel(const K1Params p) {
    griddep_launch_dependents();
    const int row = row_of_position(p, blockIdx.x, threadIdx.x & 31);
    griddep_wait();
    quantize_row_regs<NT, 0, NV, XOP>(p, blockIdx.x, row, threadIdx.x);
}

// The MXFP4 base's form of it: a block of 32 elements is all its quantization needs, so a warp takes 1024 elements of a row at a time --
// four loads per lane (and, with the input transform, four more) in flight -- and walks the batch with the grid's stride; the segment
// index is read once per warp.  Bound by memory (x read, codes and sorted copy written: 4.5 bytes per element), with the transform by its
// instructions; the plain form spills 16 bytes under its bound of six CTAs.  Whole launch, against a CTA per row: 8192 rows of 4096
// 37 -> 29-33 us; SiLU * mul, 2048 rows of 12288 45 -> 41.
template <int XOP>
__global__ void __launch_bounds__(kK1Threads, XOP == OB_X_SILU_MUL ? 4 : 6) k1_quant_mx_kernel(const K1Params p) {
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int chunks = (p.K + 1023) >> 10, groups = p.K >> 3;
    const int stride = gridDim.x * (kK1Threads / 32);
    const int total = p.M * chunks;
    int n_all, n_ad;
    segment_totals(p.meta, p.L, lane, n_all, n_ad);
    n_all = min(n_all, p.M);
    griddep_wait();
    for (int u = blockIdx.x * (kK1Threads / 32) + (threadIdx.x >> 5); u < total; u += stride) {
        const int pos = u / chunks, c = u - pos * chunks;
        const __nv_bfloat16* xr = p.x + (int64_t)position_row(p.meta, pos, p.M, n_all, n_ad) * p.ldx;
        uint4 x[4];
        __nv_bfloat162 lo = __floats2bfloat162_rn(0.0f, 0.0f), hi = lo;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = c * 128 + q * 32 + lane;
            if (XOP == OB_X_SILU_MUL) x[q] = i < groups ? silu_mul8_quick(p, xr, i * 8, lo, hi) : make_uint4(0u, 0u, 0u, 0u);
            else x[q] = i < groups ? __ldg(reinterpret_cast<const uint4*>(xr) + i) : make_uint4(0u, 0u, 0u, 0u);
        }
        if (XOP == OB_X_SILU_MUL && silu_quick_left_range(lo, hi)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = (c * 128 + q * 32 + lane) * 8;
                if (k < p.K) x[q] = silu_mul8_plain(xr + k, xr + p.K + k);
            }
        }
        uint32_t* out = reinterpret_cast<uint32_t*>(p.xq + (size_t)pos * (size_t)(p.K >> 1));
        uint4* xo = reinterpret_cast<uint4*>(p.xs + (size_t)pos * (size_t)p.K);
        // the lane's block of group q: K slot 4 c + q, within it block lane / 4 -- MMA pair lane / 16, scale (lane / 4) % 4
        uint8_t* sf = mx_scale_slot(p, pos, c * 32) + ((lane >> 4) & 1) * 512 + ((lane >> 2) & 3);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = c * 128 + q * 32 + lane;
            float v[8];
            unpack8(x[q], v);
            uint32_t byte;
            const uint32_t codes = mx_quantize8(v, byte);
            if (i < groups) {
                xo[i] = x[q];
                out[i] = codes;
            }
            if ((lane & 3) == 0 && c * 4 + q < p.kslots) sf[(size_t)q * p.nblk * sf_slot_bytes(OB_BASE_MXFP4)] = (uint8_t)byte;
        }
    }
}

// `carve`: leave the SMs configured for the largest shared-memory carve-out.  The split between it and the first-level cache
// only changes on an idle SM, and with the default one the dependent shrink's CTAs (194 KB each) cannot start -- read the segment
// index, request their first A tiles -- before this launch has drained: gate_up, K1 at 200 tokens 29 -> 26.5 us, at 8192 77 -> 78.
// Not for the longer rows: their kernels spill a few registers into that cache (down, K1 at 2048 tokens 86 -> 98).
template <int NT, typename Kernel>
static cudaError_t launch_quant_kernel(cudaLaunchConfig_t cfg, const K1Params& p, Kernel kernel, std::atomic<unsigned long long>* carve) {
    int dev = 0;
    if (carve != nullptr && cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 && !(carve->load() & (1ull << dev))) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return e;
        carve->fetch_or(1ull << dev);
    }
    cfg.blockDim = dim3(NT);
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int BASE, int XOP>
static cudaError_t launch_quant_only(const cudaLaunchConfig_t& cfg, const K1Params& p) {
    static std::atomic<unsigned long long> carved{0};
    if constexpr (BASE == OB_BASE_FP8 && XOP != OB_X_QUANTIZED) {
        if (p.K <= 8 * 2 * 256) return launch_quant_kernel<256>(cfg, p, k1_quant_regs_kernel<256, 2, XOP, XOP == OB_X_SILU_MUL ? 4 : 8>, &carved);
        // (with the transform 512 threads measured 4 us less at 200 rows of 12288, 2 us at 2048; without it they are equal)
        if constexpr (XOP == OB_X_SILU_MUL) {
            if (p.K <= 8 * 3 * 512) return launch_quant_kernel<512>(cfg, p, k1_quant_regs_kernel<512, 3, OB_X_SILU_MUL, 2>, nullptr);
        } else {
            if (p.K <= 8 * 6 * 256) return launch_quant_kernel<256>(cfg, p, k1_quant_regs_kernel<256, 6, OB_X_PLAIN, 4>, nullptr);
        }
    }
    if constexpr (BASE == OB_BASE_MXFP4 && XOP != OB_X_QUANTIZED) {
        cudaLaunchConfig_t wide = cfg;
        const long long ctas = ((long long)p.M * ((p.K + 1023) / 1024) + kK1Threads / 32 - 1) / (kK1Threads / 32);
        const long long most = 148LL * (XOP == OB_X_SILU_MUL ? 4 : 6);
        wide.gridDim = dim3((unsigned)(ctas < most ? ctas : most));
        return launch_quant_kernel<kK1Threads>(wide, p, k1_quant_mx_kernel<XOP>, &carved);
    } else {
        return launch_quant_kernel<kK1Threads>(cfg, p, k1_quant_kernel<BASE, XOP>, nullptr);
    }
}

template <int LORA_FMT, int BASE>
static cudaError_t launch_k1_impl(const K1Params& p, int grid, int pdl, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kK1Threads);
    cfg.dynamicSmemBytes = 0;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    if constexpr (BASE != OB_BASE_MXFP4) {
        if (p.looped) {
            // Beside the persistent GEMM, K1 needs next to no shared memory but must leave the SMs it runs on configured for the
            // LARGEST shared-memory carve-out: the split between L1 and shared memory only changes on an idle SM, so with the
            // default (small) carve-out the dependent GEMM's CTAs (150-200 KB each) could not become resident beside K1's and
            // the two kernels of the chain would run one after the other.  (It costs this form most of its L1 cache.)
            static std::atomic<unsigned long long> carved{0};
            int dev = 0;
            if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 && !(carved.load() & (1ull << dev))) {
                cudaError_t e = cudaFuncSetAttribute(k1_kernel<LORA_FMT, BASE, true, OB_X_PLAIN>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                                     (int)cudaSharedmemCarveoutMaxShared);
                if (e != cudaSuccess) return e;
                carved.fetch_or(1ull << dev);
            }
            return cudaLaunchKernelEx(&cfg, k1_kernel<LORA_FMT, BASE, true, OB_X_PLAIN>, p);
        }
    }
    // no shrink warps in this launch (the tensor-core shrink follows: the sorted copy of x is wanted).  SiLU * mul at 2048
    // rows of 12288: 127 us in k1_kernel<XOP> (two CTAs per SM, the transform evaluated three times)
    const bool quant_only = grid == p.n_quant_ctas && p.xs != nullptr && p.xq_ready == nullptr && p.trace == nullptr;
    if constexpr (BASE != OB_BASE_NVFP4) {
        if (p.x_op == OB_X_QUANTIZED)
            return quant_only ? launch_quant_only<BASE, OB_X_QUANTIZED>(cfg, p)
                              : cudaLaunchKernelEx(&cfg, k1_kernel<LORA_FMT, BASE, false, OB_X_QUANTIZED>, p);
    }
    if (quant_only)
        return p.x_op != OB_X_PLAIN ? launch_quant_only<BASE, OB_X_SILU_MUL>(cfg, p) : launch_quant_only<BASE, OB_X_PLAIN>(cfg, p);
    if (p.x_op != OB_X_PLAIN) return cudaLaunchKernelEx(&cfg, k1_kernel<LORA_FMT, BASE, false, OB_X_SILU_MUL>, p);
    return cudaLaunchKernelEx(&cfg, k1_kernel<LORA_FMT, BASE, false, OB_X_PLAIN>, p);
}

template <int LORA_FMT>
static cudaError_t launch_k1_base(const K1Params& p, int grid, int pdl, cudaStream_t stream) {
    return p.base_fmt == OB_BASE_NVFP4   ? launch_k1_impl<LORA_FMT, OB_BASE_NVFP4>(p, grid, pdl, stream)
           : p.base_fmt == OB_BASE_MXFP4 ? launch_k1_impl<LORA_FMT, OB_BASE_MXFP4>(p, grid, pdl, stream)
                                         : launch_k1_impl<LORA_FMT, OB_BASE_FP8>(p, grid, pdl, stream);
}

cudaError_t launch_k1_fp8(const K1Params& p, int grid, int pdl, cudaStream_t stream) {
    switch (p.lora_fmt) {
        case kLoraFp8: return launch_k1_base<kLoraFp8>(p, grid, pdl, stream);
        case kLoraNvfp4: return launch_k1_base<kLoraNvfp4>(p, grid, pdl, stream);
        default: return launch_k1_base<kLoraBf16>(p, grid, pdl, stream);
    }
}

}  // namespace ob
