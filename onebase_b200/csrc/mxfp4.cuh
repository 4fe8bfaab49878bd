// MXFP4 arithmetic (OCP microscaling: e2m1 elements, one power-of-two scale per 32 of them), shared by the quantizers and by
// the kernels that read the format.
//
// A block's scale is 2^e with e = floor(log2 max|v|) - 2 (2 = the exponent of e2m1's largest value, 6 = 1.5 * 2^2), stored as the
// byte e + 127; an element is the e2m1 value next to v / 2^e (ties to even, saturating at 6).  Both steps are exact
// arithmetic on fp32: the exponent is a field of max|v|'s bits and the division is a product with a power of two.  A block of zeros or of
// values below 2^-125 has byte 0 (2^-127); a block that holds an infinity or a NaN has byte 255, the format's NaN, and codes 0.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace ob {

// Bits of |v|: as integers they order like the magnitudes, infinity above every number and NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Scale byte of a block from the largest abs_bits of its elements.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// 2^(127 - byte): what an element is multiplied by before it is rounded (bytes 0 .. 252).
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127): what a code's value is multiplied by (byte 0: 2^-127, a subnormal; 255: NaN).
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7FC00000u : byte == 0u ? 0x00400000u : byte << 23);
}

// Eight values -> eight e2m1 codes, element i in bits 4i .. 4i+3: round to nearest even, saturating at +-6.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n"
        ".reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};\n"
        "}\n"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// The other way: eight codes -> their values.
__device__ __forceinline__ void e2m1x8_values(uint32_t codes, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n"
        ".reg .b8 a, b, c, d;\n"
        "mov.b32 {a, b, c, d}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n"
        "}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// The four lanes of a block (lane & 3 = its eighths pair, eight elements each) turn their elements into codes; `byte` is the
// block's scale byte in all four.  Every lane of the warp calls it.
__device__ __forceinline__ uint32_t mx_quantize8(const float (&v)[8], uint32_t& byte) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[i]));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    byte = mx_scale_byte(top);
    const float inv = mx_inverse(byte);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = v[i] * inv;
    return byte == 255u ? 0u : e2m1x8(q);
}

}  // namespace ob
