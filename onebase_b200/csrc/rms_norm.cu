// Root-mean-square norm with the residual's addition in front and an output in 8 or 4 bits behind:
//
//   s = x + residual                      (fp32; residual_out = s rounded once)
//   y = (s w) / sqrt(mean(s^2) + eps)     (fp32; y's store rounds once)
//   FP8:   scale = max(max|y| / 448, 1 / (448 * 512)) per row, codes = e4m3(y / scale)
//   MXFP4: per 32 elements, see mxfp4.cuh
//
// The codes are rounded from the fp32 y and not from its 16-bit store: one rounding instead of two, and a scale that does not jump
// with the store's last bit.  max|y| needs no second pass over the row: rounding and the product with a positive number are
// monotone, so max|y| = max|s w| / sqrt(..) and both reductions run together.
//
// A NaN (or an infinity) in a row makes its sum of squares one, and with it every y, the scale and every code of the row.
#include <type_traits>

#include "mxfp4.cuh"
#include "ob_common.cuh"
#include "ob_ptx.cuh"

namespace ob {

constexpr int kNormThreads = 256;
constexpr float kNormFp8Max = 448.0f, kNormMinScale = 1.0f / (448.0f * 512.0f);   // the floor of the FP8 projection's token scales

template <typename T>
__device__ __forceinline__ float to_f(T v) {
    if constexpr (std::is_same_v<T, __half>) return __half2float(v);
    else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v) {
    if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

struct NormRow {                // where row (token m, head h) lies
    const uint8_t* x;
    const uint8_t* r;
    uint8_t* ro;
    uint8_t* y;
};
__device__ __forceinline__ NormRow norm_row(const ObRmsNorm& p, long long row) {
    const long long m = p.H == 1 ? row : row / p.H, h = p.H == 1 ? 0 : row - m * p.H;
    NormRow a;
    a.x = static_cast<const uint8_t*>(p.x) + (m * p.x_ld + h * p.x_hd) * 2;
    a.r = p.residual ? static_cast<const uint8_t*>(p.residual) + (m * p.residual_ld + h * p.residual_hd) * 2 : nullptr;
    a.ro = p.residual_out ? static_cast<uint8_t*>(p.residual_out) + (m * p.residual_out_ld + h * p.residual_out_hd) * 2 : nullptr;
    a.y = p.y ? static_cast<uint8_t*>(p.y) + (m * p.y_ld + h * p.y_hd) * 2 : nullptr;
    return a;
}

// scale of an FP8 row; a NaN stays one (fmaxf would drop it)
__device__ __forceinline__ float norm_fp8_scale(float amax) {
    const float sc = __fdiv_rn(amax, kNormFp8Max);
    return sc < kNormMinScale ? kNormMinScale : sc;
}

// Any row: one CTA reads it twice, element by element.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) rms_norm_any_kernel(const ObRmsNorm p) {
    griddep_launch_dependents();
    __shared__ float s_sum[kNormThreads / 32], s_max[kNormThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x;
    const NormRow a = norm_row(p, row);
    const T* x = reinterpret_cast<const T*>(a.x);
    const T* r = reinterpret_cast<const T*>(a.r);
    const bool w32 = p.weight_dtype == OB_DTYPE_F32;
    griddep_wait();
    auto value = [&](int i) { return r ? to_f(x[i]) + to_f(r[i]) : to_f(x[i]); };
    auto weight = [&](int i) { return !p.weight ? 1.0f : w32 ? static_cast<const float*>(p.weight)[i] : to_f(static_cast<const T*>(p.weight)[i]); };
    float sum = 0.0f, top = 0.0f;
    for (int i = tid; i < p.K; i += kNormThreads) {
        const float s = value(i);
        sum = fmaf(s, s, sum);
        top = fmaxf(top, fabsf(s * weight(i)));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (lane == 0) { s_sum[warp] = sum; s_max[warp] = top; }
    __syncthreads();
    sum = s_sum[0];
    top = s_max[0];
#pragma unroll
    for (int w = 1; w < kNormThreads / 32; ++w) { sum += s_sum[w]; top = fmaxf(top, s_max[w]); }
    const float rstd = __frcp_rn(__fsqrt_rn(__fdiv_rn(sum, (float)p.K) + p.eps));
    const float sc = norm_fp8_scale(top * rstd);
    if (p.quant == OB_QUANT_FP8 && tid == 0) static_cast<float*>(p.scales)[row] = sc;
    for (int i = tid; i < p.K; i += kNormThreads) {
        const float s = value(i), y = s * weight(i) * rstd;
        if (a.ro) reinterpret_cast<T*>(a.ro)[i] = from_f<T>(s);
        if (a.y) reinterpret_cast<T*>(a.y)[i] = from_f<T>(y);
        if (p.quant == OB_QUANT_FP8) {
            static_cast<uint8_t*>(p.codes)[row * p.K + i] = (uint8_t)(cvt_e4m3x2(__fdiv_rn(y, sc), 0.0f) & 0xFFu);
        } else if (p.quant == OB_QUANT_MXFP4) {       // K % 32 == 0: a warp's lanes are one block's elements
            uint32_t t = abs_bits(y);
#pragma unroll
            for (int o = 16; o; o >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
            const uint32_t byte = mx_scale_byte(t);
            const float q = y * mx_inverse(byte), next = __shfl_down_sync(0xffffffffu, q, 1);
            const float v[8] = {q, next, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if ((lane & 1) == 0) static_cast<uint8_t*>(p.codes)[(row * p.K + i) >> 1] = byte == 255u ? 0 : (uint8_t)(e2m1x8(v) & 0xFFu);
            if (lane == 0) static_cast<uint8_t*>(p.scales)[(row * p.K + i) >> 5] = (uint8_t)byte;
        }
    }
}

// Rows that take 16-byte accesses: G threads hold one row in registers, NV groups of eight elements each, so that every tensor crosses
// memory once.  Up to 32 threads a row is a part of one warp and needs no barrier; above, one.  The new residual stream is stored as
// soon as it is formed and only s w is kept across the reduction.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[8]) {
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
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[8]) {
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
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__host__ __device__ constexpr int norm_block(int G) { return G < 128 ? 128 : G; }

template <typename T, int Q, int G, int NV>
__global__ void __launch_bounds__(norm_block(G)) rms_norm_rows_kernel(const ObRmsNorm p) {
    griddep_launch_dependents();
    constexpr int kRows = norm_block(G) / G;          // rows of a CTA
    const int t = threadIdx.x % G;
    const long long row = (long long)blockIdx.x * kRows + threadIdx.x / G;
    const bool live = kRows == 1 || row < (long long)p.M * p.H;
    const NormRow a = norm_row(p, live ? row : 0);
    const int nvec = live ? p.K >> 3 : 0;
    const bool w32 = p.weight_dtype == OB_DTYPE_F32;
    griddep_wait();
    uint4 xv[NV], rv[NV];
    float s[NV][8];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int i = t + q * G;
        xv[q] = i < nvec ? reinterpret_cast<const uint4*>(a.x)[i] : make_uint4(0u, 0u, 0u, 0u);
        rv[q] = a.r && i < nvec ? reinterpret_cast<const uint4*>(a.r)[i] : make_uint4(0u, 0u, 0u, 0u);
    }
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int i = t + q * G;
        unpack16<T>(xv[q], s[q]);
        if (a.r) {
            float r[8];
            unpack16<T>(rv[q], r);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[q][e] += r[e];
        }
        if (a.ro && i < nvec) reinterpret_cast<uint4*>(a.ro)[i] = pack16<T>(s[q]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(s[q][e], s[q][e], sum);
        if (p.weight && i < nvec) {
            float w[8];
            if (w32) {
                const float4 lo = __ldg(static_cast<const float4*>(p.weight) + 2 * i), hi = __ldg(static_cast<const float4*>(p.weight) + 2 * i + 1);
                w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w; w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w;
            } else {
                unpack16<T>(__ldg(static_cast<const uint4*>(p.weight) + i), w);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s[q][e] *= w[e];
        }
        if (Q == OB_QUANT_FP8)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(s[q][e]));
    }
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (Q == OB_QUANT_FP8) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if constexpr (G > 32) {
        constexpr int kWarps = G / 32;
        __shared__ float s_sum[kWarps], s_max[kWarps];
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0) {
            s_sum[warp] = sum;
            if (Q == OB_QUANT_FP8) s_max[warp] = top;
        }
        __syncthreads();
        sum = s_sum[lane % kWarps];                   // (kWarps is a power of two: the shuffles below stay within the copies)
        top = Q == OB_QUANT_FP8 ? s_max[lane % kWarps] : 0.0f;
#pragma unroll
        for (int o = kWarps / 2; o; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (Q == OB_QUANT_FP8) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
    }
    const float rstd = __frcp_rn(__fsqrt_rn(__fdiv_rn(sum, (float)p.K) + p.eps));
    const float sc = Q == OB_QUANT_FP8 ? norm_fp8_scale(top * rstd) : 0.0f;
    if (Q == OB_QUANT_FP8 && t == 0 && live) static_cast<float*>(p.scales)[row] = sc;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int i = t + q * G;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[q][e] *= rstd;
        if (a.y && i < nvec) reinterpret_cast<uint4*>(a.y)[i] = pack16<T>(s[q]);
        if (Q == OB_QUANT_FP8) {
            if (i < nvec) {
                uint32_t c[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] = cvt_e4m3x2(__fdiv_rn(s[q][2 * e], sc), __fdiv_rn(s[q][2 * e + 1], sc));
                reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.codes) + row * p.K)[i] = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
            }
        } else if (Q == OB_QUANT_MXFP4) {             // (K % 32 == 0: the four lanes of a block are all in the row, or none is)
            uint32_t byte;
            const uint32_t c = mx_quantize8(s[q], byte);
            if (i < nvec) {
                reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.codes) + row * (p.K >> 1))[i] = c;
                if ((i & 3) == 0) static_cast<uint8_t*>(p.scales)[row * (p.K >> 5) + (i >> 2)] = (uint8_t)byte;
            }
        }
    }
}

template <typename Kernel>
static cudaError_t launch_norm(const ObRmsNorm& p, Kernel kernel, long long ctas, int threads, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int Q, int G, int NV>
static cudaError_t launch_rows(const ObRmsNorm& p, cudaStream_t stream) {
    constexpr int kRows = norm_block(G) / G;
    return launch_norm(p, rms_norm_rows_kernel<T, Q, G, NV>, ((long long)p.M * p.H + kRows - 1) / kRows, norm_block(G), stream);
}

// Threads per row: as many groups of eight as keep a few loads of a thread in flight; few rows take twice the threads of one load each.
template <typename T, int Q>
static cudaError_t launch_rows_of(const ObRmsNorm& p, cudaStream_t stream) {
    const long long rows = (long long)p.M * p.H;
    if (p.K <= 128) return launch_rows<T, Q, 16, 1>(p, stream);
    if (p.K <= 256) return launch_rows<T, Q, 32, 1>(p, stream);
    if (p.K <= 512) return launch_rows<T, Q, 32, 2>(p, stream);
    if (p.K <= 1024) return launch_rows<T, Q, 32, 4>(p, stream);
    if (p.K <= 2048) return launch_rows<T, Q, 128, 2>(p, stream);
    if (p.K <= 4096 && rows <= 296) return launch_rows<T, Q, 512, 1>(p, stream);
    if (p.K <= 4096) return launch_rows<T, Q, 256, 2>(p, stream);
    if (p.K <= 8192) return launch_rows<T, Q, 512, 2>(p, stream);
    if (p.K <= 16384) return launch_rows<T, Q, 512, 4>(p, stream);
    return launch_rows<T, Q, 1024, 4>(p, stream);
}

template <typename T>
static cudaError_t launch_typed(const ObRmsNorm& p, cudaStream_t stream) {
    auto whole = [&](const void* ptr, int64_t ld, int64_t hd) {      // 16-byte accesses at every row
        return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && (ptr == nullptr || (ld % 8 == 0 && (p.H == 1 || hd % 8 == 0)));
    };
    const bool rows = p.K % 8 == 0 && p.K <= 32768 && whole(p.x, p.x_ld, p.x_hd) && whole(p.residual, p.residual_ld, p.residual_hd) &&
                      whole(p.residual_out, p.residual_out_ld, p.residual_out_hd) && whole(p.y, p.y_ld, p.y_hd) && whole(p.weight, 0, 0);
    if (!rows) return launch_norm(p, rms_norm_any_kernel<T>, (long long)p.M * p.H, kNormThreads, stream);
    return p.quant == OB_QUANT_FP8     ? launch_rows_of<T, OB_QUANT_FP8>(p, stream)
           : p.quant == OB_QUANT_MXFP4 ? launch_rows_of<T, OB_QUANT_MXFP4>(p, stream)
                                       : launch_rows_of<T, OB_QUANT_NONE>(p, stream);
}

cudaError_t launch_rms_norm(const ObRmsNorm& p, cudaStream_t stream) {
    return p.dtype == OB_DTYPE_F16 ? launch_typed<__half>(p, stream) : launch_typed<__nv_bfloat16>(p, stream);
}

}  // namespace ob
