// Device helpers of the 8-bit key/value cache: power-of-two scales and E4M3 conversions.
//
// A scale is the smallest power of two 2^e, e >= -126, with largest <= 448 * 2^e.  E4M3 is a floating format: its relative
// precision does not depend on where in its range a value lies, so a scale only has to place that range, and a power of two
// does so without a rounding of its own.  x / 2^e is exact, raising a scale re-rounds only codes that become subnormal, and
// code * 2^e is exact in f32, and in bf16 from e = -124 on (below, subnormal codes are off by 2^-134 at most).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace lfm25 {

constexpr int32_t kLeastScaleExponent = -126;

// e for the bits of a finite, non-negative f32: 448 = 1.75 * 2^8
__device__ __forceinline__ int32_t scale_exponent(uint32_t largest_bits) {
    const int32_t exponent = static_cast<int32_t>(largest_bits >> 23) - 127 - 8 + ((largest_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(exponent, kLeastScaleExponent);
}

// The scale that a page goes on with.  What is no number in 2^-126 .. 2^120 (an arena that was never written, stray bits) counts as the
// least; a number in between that is no power of two, which no append leaves, is taken as it is.
__device__ __forceinline__ float stored_scale(float scale) {
    return scale >= 1.1754944e-38f && scale <= 1.329228e36f ? scale : 1.1754944e-38f;
}

// least e with scale <= 2^e
__device__ __forceinline__ int32_t exponent_above(float scale) {
    const uint32_t bits = __float_as_uint(scale);
    return static_cast<int32_t>(bits >> 23) - 127 + ((bits & 0x7fffffu) != 0 ? 1 : 0);
}

// 2^e for -126 <= e <= 127; below that 0, as the product with a code rounds to 0 there anyway
__device__ __forceinline__ float power_of_two(int32_t e) {
    return e < -126 ? 0.0f : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// two E4M3 codes -> f16x2 (exact; NaN stays NaN)
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
    uint32_t halves;
    asm("{\n.reg .b16 low;\nmov.b32 {low, _}, %1;\ncvt.rn.f16x2.e4m3x2 %0, low;\n}" : "=r"(halves) : "r"(codes));
    return halves;
}
__device__ __forceinline__ uint32_t e4m3x2_high_to_f16x2(uint32_t codes) {
    uint32_t halves;
    asm("{\n.reg .b16 high;\nmov.b32 {_, high}, %1;\ncvt.rn.f16x2.e4m3x2 %0, high;\n}" : "=r"(halves) : "r"(codes));
    return halves;
}
__device__ __forceinline__ float2 f16x2_to_float2(uint32_t halves) {
    return __half22float2(*reinterpret_cast<const __half2*>(&halves));
}

__device__ __forceinline__ uint32_t pack_f16x2(float low, float high) {
    const __half2 pair = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&pair);
}

__device__ __forceinline__ float2 bf16x2_to_float2(uint32_t pair) {
    return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
}

// a * b + c for two values at a time, b the same for both
__device__ __forceinline__ float2 fma_pair(float2 a, float b, float2 c) {
    float2 out;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %4};\nmov.b64 z, {%5, %6};\nfma.rn.f32x2 x, x, y, z;\n"
        "mov.b64 {%0, %1}, x;\n}"
        : "=f"(out.x), "=f"(out.y) : "f"(a.x), "f"(a.y), "f"(b), "f"(c.x), "f"(c.y));
    return out;
}

// D(16x8, f32) += A(16x16, f16, row) * B(16x8, f16, col)
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D(16x8, f32) = A(16x16, f16, row) * B(16x8, f16, col)
__device__ __forceinline__ void mma_f16_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                    uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

}  // namespace lfm25
