// MXFP4 quantization and its inverse on whole tensors (see mxfp4.cuh for the format and the rounding).
//
// Four lanes own one block of 32 elements, eight each: a lane loads 16 bytes of a 16-bit tensor (32 of fp32), the block's largest
// magnitude takes two shuffles, and a lane stores its eight codes as one 32-bit word.  Both directions are bound by memory: 2 bytes
// read and 17/32 written per bf16 element, or the reverse.  What they write may be a projection's weight or adapter, which are read
// before the wait on the preceding kernel: such a write is followed by ob_operand_fence (leaving out the early trigger would not do,
// as a dependent may also start when the CTAs have left).
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

// Where group i of eight elements lies: dense tensors are one long row (no division); else row i / vpr, in 32 bits while they suffice.
template <bool DENSE>
__device__ __forceinline__ long long mx_offset(long long i, long long total, int vpr, long long ld) {
    if (DENSE) return i * 8;
    const long long row = total <= 0xFFFFFFFFll ? (long long)((uint32_t)i / (uint32_t)vpr) : i / vpr;
    return row * ld + (i - row * vpr) * 8;
}

template <typename T, bool VEC, bool DENSE, int U>
__global__ void __launch_bounds__(kMxThreads)
mxfp4_quantize_kernel(const T* __restrict__ x, long long total, int vpr, long long ldx, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    griddep_wait();
    const long long i0 = (long long)blockIdx.x * (kMxThreads * U) + threadIdx.x;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {                     // (the four lanes of a block are all in range, or none is)
        const long long i = i0 + u * kMxThreads;
        if (i < total) mx_load8<T, VEC>(x + mx_offset<DENSE>(i, total, vpr, ldx), v[u]);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = i0 + u * kMxThreads;
        uint32_t byte;
        const uint32_t c = mx_quantize8(v[u], byte);
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

template <typename T, bool VEC, bool DENSE, int U>
__global__ void __launch_bounds__(kMxThreads)
mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, long long total, int vpr, T* __restrict__ out, long long ldo) {
    griddep_wait();
    const long long i0 = (long long)blockIdx.x * (kMxThreads * U) + threadIdx.x;
    uint32_t c[U], byte[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = i0 + u * kMxThreads;
        c[u] = i < total ? __ldg(codes + i) : 0u;
        byte[u] = i < total ? __ldg(scales + (i >> 2)) : 0u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = i0 + u * kMxThreads;
        float v[8];
        e2m1x8_values(c[u], v);
        const float sc = mx_scale(byte[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= sc;
        if (i < total) mx_store8<T, VEC>(out + mx_offset<DENSE>(i, total, vpr, ldo), v);
    }
}

template <typename... Params, typename... Args>
static cudaError_t mx_launch(void (*kernel)(Params...), long long total, int unroll, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    const long long per = (long long)kMxThreads * unroll, ctas = (total + per - 1) / per;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kMxThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Tensors that fill the GPU take four groups per thread (their loads in flight together), smaller ones one.
static bool mx_large(long long total) { return total > 148LL * 2048 * 4; }

template <typename T, bool VEC, bool DENSE>
static cudaError_t quantize_form(const T* x, long long total, int vpr, long long ldx, uint32_t* codes, uint8_t* scales, cudaStream_t stream) {
    return mx_large(total) ? mx_launch(mxfp4_quantize_kernel<T, VEC, DENSE, 4>, total, 4, stream, x, total, vpr, ldx, codes, scales)
                           : mx_launch(mxfp4_quantize_kernel<T, VEC, DENSE, 1>, total, 1, stream, x, total, vpr, ldx, codes, scales);
}

template <typename T>
static cudaError_t quantize_typed(const void* xp, long long rows, int K, long long ldx, void* codes, void* scales, cudaStream_t stream) {
    const T* x = static_cast<const T*>(xp);
    uint32_t* c = static_cast<uint32_t*>(codes);
    uint8_t* s = static_cast<uint8_t*>(scales);
    const int vpr = K >> 3;
    const long long total = rows * vpr;
    if ((reinterpret_cast<uintptr_t>(xp) & 15u) != 0 || (rows > 1 && (ldx * (long long)sizeof(T)) % 16 != 0))
        return quantize_form<T, false, false>(x, total, vpr, ldx, c, s, stream);
    return rows == 1 || ldx == K ? quantize_form<T, true, true>(x, total, vpr, ldx, c, s, stream)
                                 : quantize_form<T, true, false>(x, total, vpr, ldx, c, s, stream);
}

template <typename T, bool VEC, bool DENSE>
static cudaError_t dequantize_form(const uint32_t* codes, const uint8_t* scales, long long total, int vpr, T* out, long long ldo, cudaStream_t stream) {
    return mx_large(total) ? mx_launch(mxfp4_dequantize_kernel<T, VEC, DENSE, 4>, total, 4, stream, codes, scales, total, vpr, out, ldo)
                           : mx_launch(mxfp4_dequantize_kernel<T, VEC, DENSE, 1>, total, 1, stream, codes, scales, total, vpr, out, ldo);
}

template <typename T>
static cudaError_t dequantize_typed(const void* codes, const void* scales, long long rows, int K, void* outp, long long ldo, cudaStream_t stream) {
    const uint32_t* c = static_cast<const uint32_t*>(codes);
    const uint8_t* s = static_cast<const uint8_t*>(scales);
    T* out = static_cast<T*>(outp);
    const int vpr = K >> 3;
    const long long total = rows * vpr;
    if ((reinterpret_cast<uintptr_t>(outp) & 15u) != 0 || (rows > 1 && (ldo * (long long)sizeof(T)) % 16 != 0))
        return dequantize_form<T, false, false>(c, s, total, vpr, out, ldo, stream);
    return rows == 1 || ldo == K ? dequantize_form<T, true, true>(c, s, total, vpr, out, ldo, stream)
                                 : dequantize_form<T, true, false>(c, s, total, vpr, out, ldo, stream);
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
