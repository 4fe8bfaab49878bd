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

cudaError_t launch_rms_norm(const ObRmsNorm& p, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)p.M * p.H));
    cfg.blockDim = dim3(kNormThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return p.dtype == OB_DTYPE_F16 ? cudaLaunchKernelEx(&cfg, rms_norm_any_kernel<__half>, p)
                                   : cudaLaunchKernelEx(&cfg, rms_norm_any_kernel<__nv_bfloat16>, p);
}

}  // namespace ob
