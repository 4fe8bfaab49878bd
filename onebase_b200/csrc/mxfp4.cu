// MXFP4 quantization and its inverse on whole tensors (see mxfp4.cuh for the format and the rounding).
//
// Four lanes own one block of 32 elements, eight each: a lane loads 16 bytes of a 16-bit tensor (32 of fp32), the block's largest
// magnitude takes two shuffles, and a lane stores its eight codes as one 32-bit word.  Both directions are bound by memory: 2 bytes
// read and 17/32 written per bf16 element, or the reverse.
#include <type_traits>

#include "mxfp4.cuh"
#include "ob_common.cuh"
#include "ob_ptx.cuh"

namespace ob {

constexpr int kMxThreads = 256;

template <typename T, bool VEC>
__device__ __forceinline__ void mx_load8(const T* src, float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)src[i];
    } else if constexpr (std::is_same_v<T, float>) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(src)), b = __ldg(reinterpret_cast<const float4*>(src) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(src));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x; v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]);
            }
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mxfp4_quantize_kernel(const T* __restrict__ x, long long rows, int K, long long ldx, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    griddep_launch_dependents();
    griddep_wait();
    const int vpr = K >> 3;                           // groups of eight per row, a multiple of four
    const long long total = rows * vpr;
    for (long long g = (long long)blockIdx.x * kMxThreads; g < total; g += (long long)gridDim.x * kMxThreads) {
        const long long i = g + threadIdx.x;          // (the four lanes of a block are all in range, or none is)
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (i < total) {
            const long long row = i / vpr;
            mx_load8<T, VEC>(x + row * ldx + (i - row * vpr) * 8, v);
        }
        uint32_t byte;
        const uint32_t c = mx_quantize8(v, byte);
        if (i < total) {
            codes[i] = c;
            if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
        }
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void mx_store8(T* dst, const float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = (T)v[i];
    } else if constexpr (std::is_same_v<T, float>) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, long long rows, int K, T* __restrict__ out, long long ldo) {
    griddep_launch_dependents();
    griddep_wait();
    const int vpr = K >> 3;
    const long long total = rows * vpr;
    for (long long i = (long long)blockIdx.x * kMxThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kMxThreads) {
        float v[8];
        e2m1x8_values(codes[i], v);
        const float sc = mx_scale(scales[i >> 2]);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= sc;
        const long long row = i / vpr;
        mx_store8<T, VEC>(out + row * ldo + (i - row * vpr) * 8, v);
    }
}

static cudaLaunchConfig_t mx_config(long long total, cudaStream_t stream, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    long long blocks = (total + kMxThreads - 1) / kMxThreads;
    if (blocks > (1 << 30)) blocks = 1 << 30;
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kMxThreads);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

template <typename T>
static cudaError_t quantize_typed(const void* x, long long rows, int K, long long ldx, void* codes, void* scales, cudaStream_t stream) {
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = mx_config(rows * (K >> 3), stream, attr);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (ldx * (long long)sizeof(T)) % 16 == 0;
    return vec ? cudaLaunchKernelEx(&cfg, mxfp4_quantize_kernel<T, true>, static_cast<const T*>(x), rows, K, ldx, static_cast<uint32_t*>(codes),
                                    static_cast<uint8_t*>(scales))
               : cudaLaunchKernelEx(&cfg, mxfp4_quantize_kernel<T, false>, static_cast<const T*>(x), rows, K, ldx, static_cast<uint32_t*>(codes),
                                    static_cast<uint8_t*>(scales));
}

template <typename T>
static cudaError_t dequantize_typed(const void* codes, const void* scales, long long rows, int K, void* out, long long ldo, cudaStream_t stream) {
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = mx_config(rows * (K >> 3), stream, attr);
    const bool vec = (reinterpret_cast<uintptr_t>(out) & 15u) == 0 && (ldo * (long long)sizeof(T)) % 16 == 0;
    return vec ? cudaLaunchKernelEx(&cfg, mxfp4_dequantize_kernel<T, true>, static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(scales),
                                    rows, K, static_cast<T*>(out), ldo)
               : cudaLaunchKernelEx(&cfg, mxfp4_dequantize_kernel<T, false>, static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(scales),
                                    rows, K, static_cast<T*>(out), ldo);
}

cudaError_t launch_mxfp4_quantize(const void* x, int dtype, long long rows, int K, long long ldx, void* codes, void* scales, cudaStream_t stream) {
    return dtype == OB_DTYPE_F32   ? quantize_typed<float>(x, rows, K, ldx, codes, scales, stream)
           : dtype == OB_DTYPE_F16 ? quantize_typed<__half>(x, rows, K, ldx, codes, scales, stream)
                                   : quantize_typed<__nv_bfloat16>(x, rows, K, ldx, codes, scales, stream);
}

cudaError_t launch_mxfp4_dequantize(const void* codes, const void* scales, int dtype, long long rows, int K, void* out, long long ldo,
                                    cudaStream_t stream) {
    return dtype == OB_DTYPE_F32   ? dequantize_typed<float>(codes, scales, rows, K, out, ldo, stream)
           : dtype == OB_DTYPE_F16 ? dequantize_typed<__half>(codes, scales, rows, K, out, ldo, stream)
                                   : dequantize_typed<__nv_bfloat16>(codes, scales, rows, K, out, ldo, stream);
}

}  // namespace ob
