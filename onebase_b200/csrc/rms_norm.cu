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
// A NaN in a row makes every y, the scale and every code of the row one.  An infinity makes 1 / sqrt(..) zero: the row's y is NaN there and
// 0 elsewhere, an FP8 row's scale and codes are NaN.
#include <type_traits>

#include "mxfp4.cuh"
#include "ob_common.cuh"
#include "ob_ptx.cuh"

namespace ob {

__host__ __device__ constexpr int norm_block(int G) { return G < 64 ? 128 : G; }   // threads of a CTA: several short rows share one
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

// y / scale from the rounded inv = 1 / scale: the product, corrected by its own remainder (Markstein), which is the quotient rounded once
// -- as the projection's own quantizer divides -- in two more instructions instead of a division's dozen.  The product alone is off by a last
// bit for a fifth of all y, and where y / scale is a tie of e4m3 that gave another code.
__device__ __forceinline__ float norm_quotient(float y, float sc, float inv) {
    const float q = y * inv;
    return fmaf(-fmaf(q, sc, -y), inv, q);            // (in this form a zero keeps its sign)
}

// Sum and (FP8) largest magnitude over the G threads of a row.
template <int G, bool MAX>
__device__ __forceinline__ void norm_reduce(float& sum, float& top) {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (MAX) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if constexpr (G > 32) {                           // (one row per CTA)
        constexpr int kWarps = G / 32;
        __shared__ float s_sum[kWarps], s_max[kWarps];
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0) {
            s_sum[warp] = sum;
            if (MAX) s_max[warp] = top;
        }
        __syncthreads();
        sum = s_sum[lane % kWarps];                   // (kWarps is a power of two: the shuffles below stay within the copies)
        if (MAX) top = s_max[lane % kWarps];
#pragma unroll
        for (int o = kWarps / 2; o; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (MAX) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
    }
}
__device__ __forceinline__ float norm_rstd(float sum, const ObRmsNorm& p) { return __frcp_rn(__fsqrt_rn(__fdiv_rn(sum, (float)p.K) + p.eps)); }

// Any row, element by element: G threads, NE elements each held in registers (NE = 0: the row is read twice instead).  Eight elements
// each: bound to the 32 registers that let an SM have its 2048 threads, at a spill of 8 bytes (with 34 and the bound, us: 2048 rows of 7393 --
// one CTA of 1024 threads per SM -- 89 -> 57, 4096 of 4001 64 -> 54, 8192 of 1999 59 -> 52, 8192 of 777 24 -> 22, but 300 of 4001 6.8 -> 7.5).
template <typename T, int G, int NE>
__global__ void __launch_bounds__(norm_block(G), NE == 8 && G >= 128 ? 2048 / G : 0) rms_norm_any_kernel(const ObRmsNorm p) {
    constexpr int kRows = norm_block(G) / G;
    const int t = threadIdx.x % G, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * kRows + threadIdx.x / G;
    const bool live = kRows == 1 || row < (long long)p.M * p.H;
    const NormRow a = norm_row(p, live ? row : 0);
    const int K = live ? p.K : 0;
    const T* x = reinterpret_cast<const T*>(a.x);
    const T* r = reinterpret_cast<const T*>(a.r);
    const bool w32 = p.weight_dtype == OB_DTYPE_F32;
    griddep_wait();
    griddep_launch_dependents();                      // (behind the wait: a successor may read, before its own, what a kernel before this one wrote)
    auto weight = [&](int i) { return !p.weight ? 1.0f : w32 ? __ldg(static_cast<const float*>(p.weight) + i) : to_f(static_cast<const T*>(p.weight)[i]); };
    float s[NE > 0 ? NE : 1];
    float sum = 0.0f, top = 0.0f;
    if constexpr (NE > 0) {
#pragma unroll
        for (int q = 0; q < NE; ++q) s[q] = t + q * G < K ? to_f(x[t + q * G]) : 0.0f;
        if (r) {
#pragma unroll
            for (int q = 0; q < NE; ++q) s[q] += t + q * G < K ? to_f(r[t + q * G]) : 0.0f;
        }
#pragma unroll
        for (int q = 0; q < NE; ++q) {
            const int i = t + q * G;
            if (a.ro && i < K) reinterpret_cast<T*>(a.ro)[i] = from_f<T>(s[q]);
            sum = fmaf(s[q], s[q], sum);
            s[q] *= i < K ? weight(i) : 0.0f;
            top = fmaxf(top, fabsf(s[q]));
        }
    } else {
        for (int i = t; i < K; i += G) {
            const float v = r ? to_f(x[i]) + to_f(r[i]) : to_f(x[i]);
            sum = fmaf(v, v, sum);
            top = fmaxf(top, fabsf(v * weight(i)));
        }
    }
    norm_reduce<G, true>(sum, top);
    const float rstd = norm_rstd(sum, p);
    const float sc = norm_fp8_scale(top * rstd), inv = __frcp_rn(sc);
    if (p.quant == OB_QUANT_FP8 && t == 0 && live) static_cast<float*>(p.scales)[row] = sc;
    auto store = [&](int i, float y) {                // every lane of the warp (MXFP4: K % 32 == 0, a warp's lanes are one block's elements)
        if (a.y && i < K) reinterpret_cast<T*>(a.y)[i] = from_f<T>(y);
        if (p.quant == OB_QUANT_FP8) {
            if (i < K) static_cast<uint8_t*>(p.codes)[row * p.K + i] = (uint8_t)(cvt_e4m3x2(norm_quotient(y, sc, inv), 0.0f) & 0xFFu);
        } else if (p.quant == OB_QUANT_MXFP4) {
            uint32_t m = abs_bits(y);
#pragma unroll
            for (int o = 16; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const uint32_t byte = mx_scale_byte(m);
            const float v0 = y * mx_inverse(byte), v1 = __shfl_down_sync(0xffffffffu, v0, 1);
            const float v[8] = {v0, v1, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if ((lane & 1) == 0 && i < K) static_cast<uint8_t*>(p.codes)[(row * p.K + i) >> 1] = byte == 255u ? 0 : (uint8_t)(e2m1x8(v) & 0xFFu);
            if (lane == 0 && i < K) static_cast<uint8_t*>(p.scales)[(row * p.K + i) >> 5] = (uint8_t)byte;
        }
    };
    if constexpr (NE > 0) {
#pragma unroll
        for (int q = 0; q < NE; ++q) store(t + q * G, s[q] * rstd);
    } else {
        for (int i0 = 0; i0 < K; i0 += G) {           // (whole CTAs: `store` shuffles)
            const int i = i0 + t;
            const float v = i >= K ? 0.0f : r ? to_f(x[i]) + to_f(r[i]) : to_f(x[i]);
            if (a.ro && i < K) reinterpret_cast<T*>(a.ro)[i] = from_f<T>(v);
            store(i, i < K ? v * weight(i) * rstd : 0.0f);
        }
    }
}

// Rows that take 16-byte accesses: G threads hold one row in registers, NV groups of eight elements each, so that every tensor crosses
// memory once (bound by memory: 9 bytes per element with residual and FP8 codes, 8192 rows of 4096 in 51 us, 5.9 TB/s).  Up to 32 threads a
// row is a part of one warp and needs no barrier; above, one.  The new residual stream is stored as soon as it is formed and only
// s w is kept across the reduction.
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

template <typename T, int Q, int G, int NV>
__global__ void __launch_bounds__(norm_block(G)) rms_norm_rows_kernel(const ObRmsNorm p) {
    constexpr int kRows = norm_block(G) / G;          // rows of a CTA
    const int t = threadIdx.x % G;
    const long long row = (long long)blockIdx.x * kRows + threadIdx.x / G;
    const bool live = kRows == 1 || row < (long long)p.M * p.H;
    const NormRow a = norm_row(p, live ? row : 0);
    const int nvec = live ? p.K >> 3 : 0;
    const bool w32 = p.weight_dtype == OB_DTYPE_F32;
    griddep_wait();
    griddep_launch_dependents();                      // (behind the wait, as above)
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
    norm_reduce<G, Q == OB_QUANT_FP8>(sum, top);
    const float rstd = norm_rstd(sum, p);
    const float sc = Q == OB_QUANT_FP8 ? norm_fp8_scale(top * rstd) : 0.0f, inv = Q == OB_QUANT_FP8 ? __frcp_rn(sc) : 0.0f;
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
                for (int e = 0; e < 4; ++e) c[e] = cvt_e4m3x2(norm_quotient(s[q][2 * e], sc, inv), norm_quotient(s[q][2 * e + 1], sc, inv));
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

// A thread holds four groups of eight: their loads are in flight together and small CTAs start and drain beside one another
// (8192 rows of 4096, residual and FP8 codes: 512 threads of one group 56.7 us, 256 of two 54.6, 128 of four 48.0; 8192 rows of
// 8192: 126.8, 106.8 (512 of two), 93.9 (256 of four); 262144 heads of 128: 16 threads of one 39, 8 of two 28, 4 of four 24.8).
// Inputs that do not fill the GPU wait for one row's loads, reduction and stores whatever they do, and take one group per thread (16 rows of
// 4096 3.4 -> 2.8 us, 296 4.2 -> 3.4; 592 rows 5.0 -> 5.3).
template <typename T, int Q>
static cudaError_t launch_rows_of(const ObRmsNorm& p, cudaStream_t stream) {
    if (p.K <= 128) return launch_rows<T, Q, 4, 4>(p, stream);
    if (p.K <= 256) return launch_rows<T, Q, 8, 4>(p, stream);
    const bool few = (long long)p.M * p.H * p.K <= 296 * 4096;
    if (few && p.K <= 8192) {
        if (p.K <= 512) return launch_rows<T, Q, 64, 1>(p, stream);
        if (p.K <= 1024) return launch_rows<T, Q, 128, 1>(p, stream);
        if (p.K <= 2048) return launch_rows<T, Q, 256, 1>(p, stream);
        return p.K <= 4096 ? launch_rows<T, Q, 512, 1>(p, stream) : launch_rows<T, Q, 1024, 1>(p, stream);
    }
    if (p.K <= 512) return launch_rows<T, Q, 16, 4>(p, stream);
    if (p.K <= 1024) return launch_rows<T, Q, 32, 4>(p, stream);
    if (p.K <= 2048) return launch_rows<T, Q, 64, 4>(p, stream);
    if (p.K <= 4096) return launch_rows<T, Q, 128, 4>(p, stream);
    if (p.K <= 8192) return launch_rows<T, Q, 256, 4>(p, stream);
    // (longer rows where a power of two of threads leaves a third of them idle: 8192 rows of 12288 169 us with 512 of four, 142 with 256 of
    // six; 4096 of 24576 187 with 1024 of four, 173 with 512 of six; few rows 3.9 against 4.6 the other way)
    if (p.K <= 12288 && !few) return launch_rows<T, Q, 256, 6>(p, stream);
    if (p.K <= 16384) return launch_rows<T, Q, 512, 4>(p, stream);
    return p.K <= 24576 ? launch_rows<T, Q, 512, 6>(p, stream) : launch_rows<T, Q, 1024, 4>(p, stream);
}

template <typename T, int G, int NE>
static cudaError_t launch_any(const ObRmsNorm& p, cudaStream_t stream) {
    constexpr int kRows = norm_block(G) / G;
    return launch_norm(p, rms_norm_any_kernel<T, G, NE>, ((long long)p.M * p.H + kRows - 1) / kRows, norm_block(G), stream);
}

template <typename T>
static cudaError_t launch_typed(const ObRmsNorm& p, cudaStream_t stream) {
    auto whole = [&](const void* ptr, int64_t ld, int64_t hd) {      // 16-byte accesses at every row
        return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && (ptr == nullptr || (ld % 8 == 0 && (p.H == 1 || hd % 8 == 0)));
    };
    const bool rows = p.K % 8 == 0 && p.K <= 32768 && whole(p.x, p.x_ld, p.x_hd) && whole(p.residual, p.residual_ld, p.residual_hd) &&
                      whole(p.residual_out, p.residual_out_ld, p.residual_out_hd) && whole(p.y, p.y_ld, p.y_hd) && whole(p.weight, 0, 0);
    if (!rows) {
        // eight elements per thread where they suffice: 2048 rows of 7393 57 us (256 threads reading the row twice 74), 4096 of 4001 54
        // (73), 8192 of 777 22 (42), 16 of 7393 5.1 (18).  Two bytes per access: the rows begin anywhere, and vectors would need a head and a
        // tail of their own for every tensor
        if (p.K <= 128) return launch_any<T, 32, 4>(p, stream);
        if (p.K <= 256) return launch_any<T, 32, 8>(p, stream);
        if (p.K <= 512) return launch_any<T, 64, 8>(p, stream);
        if (p.K <= 1024) return launch_any<T, 128, 8>(p, stream);
        if (p.K <= 2048) return launch_any<T, 256, 8>(p, stream);
        if (p.K <= 4096) return launch_any<T, 512, 8>(p, stream);
        if (p.K <= 8192) return launch_any<T, 1024, 8>(p, stream);
        return p.K <= 16384 ? launch_any<T, 1024, 16>(p, stream) : launch_any<T, 512, 0>(p, stream);
    }
    return p.quant == OB_QUANT_FP8     ? launch_rows_of<T, OB_QUANT_FP8>(p, stream)
           : p.quant == OB_QUANT_MXFP4 ? launch_rows_of<T, OB_QUANT_MXFP4>(p, stream)
                                       : launch_rows_of<T, OB_QUANT_NONE>(p, stream);
}

cudaError_t launch_rms_norm(const ObRmsNorm& p, cudaStream_t stream) {
    return p.dtype == OB_DTYPE_F16 ? launch_typed<__half>(p, stream) : launch_typed<__nv_bfloat16>(p, stream);
}

}  // namespace ob
