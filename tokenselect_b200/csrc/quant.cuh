// Pool rows held in 4 bits: layout and conversions shared by the kernels that write, read and attend to them.
#pragma once
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace ts {

constexpr int kQuantBlock = 16;                                // elements that share a scale

// Bytes of one (row, KV head): K codes | V codes | K scales | V scales.
template <int D>
struct QuantRow {
    static constexpr int kCodes = D / 2, kScales = D / kQuantBlock;
    static constexpr int kV = kCodes, kKScales = 2 * kCodes, kVScales = 2 * kCodes + kScales;
    static constexpr int kBytes = 2 * (kCodes + kScales);      // 9 D / 8
};

// Eight 4-bit floats (the lower half of each byte first) as pairs of fp16, exact.  `w` has to be loaded as a whole word: with a
// byte or a 16-bit load zero-extended into it, nvcc 12.9 made code that gave zeros.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
// One (the lower four bits) as fp32: its exponent and mantissa, put where fp16 has them, are the value times 2^-14.
__device__ __forceinline__ float e2m1_to_f32(uint32_t code) {
    return __half2float(__ushort_as_half((unsigned short)(((code & 8u) << 12) | ((code & 7u) << 9)))) * 16384.f;
}
// Eight values to 4-bit floats, element 2i in the lower half of byte i; nearest, ties to even, saturating at 6.
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float (&x)[8]) {
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
    return w;
}
// Two 8-bit scales (in the lower 16 bits) as fp16, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t two) {
    uint32_t h;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(two));
    return h;
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
    const uint32_t h = e4m3x2_to_f16(byte);
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}
__device__ __forceinline__ uint32_t f32_to_e4m3(float x) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
    return r & 0xffu;
}
__device__ __forceinline__ float2 half2_to_float2(uint32_t h) {
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace ts
