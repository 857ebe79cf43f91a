// Values to microscaled 4-bit codes, shared by the conversion kernels and the product that quantises its few rows itself.
#pragma once
#include "nkb_decode.cuh"

namespace nkb {

__device__ __forceinline__ uint32_t scale_byte(uint32_t largest_bits) {
    const uint32_t e = largest_bits >> 23;           // biased exponent of the largest magnitude; 255: not finite
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 1 / scale as an f32: 2^(127 - s), a normal number for every s a finite block can get (0 .. 252).
__device__ __forceinline__ float inverse_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }

// Eight values over their scale -> eight codes, value 0 in the lowest four bits.
__device__ __forceinline__ uint32_t encode8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Eight values of a 16-bit or f32 row in registers (`raw`: 16 bytes, or twice that for f32) as floats, and the bits of the largest
// magnitude. bf16: two values an instruction, since the order of magnitudes is that of their bits.
template <uint32_t kType, int kQuads>
__device__ __forceinline__ uint32_t unpack8(const uint4 (&raw)[kQuads], float (&v)[8]) {
    uint32_t largest = 0;
    if constexpr (kType == kBF16) {
        const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
        const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
        largest = max(m << 16, m & 0xffff0000u);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else {
#pragma unroll
        for (int h = 0; h < kQuads; ++h) {
            const uint32_t w[4] = {raw[h].x, raw[h].y, raw[h].z, raw[h].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (kType == kF32) v[4 * h + i] = __uint_as_float(w[i]);
                else { v[2 * i] = decode_bits<kType>(w[i] & 0xffffu); v[2 * i + 1] = decode_bits<kType>(w[i] >> 16); }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = max(largest, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    return largest;
}

// Eight values of this thread, a quarter of a block that four neighbouring threads share -> their codes and the block's scale byte.
__device__ __forceinline__ uint32_t quantise8(float (&v)[8], uint32_t largest, uint32_t &scale) {
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    scale = scale_byte(largest);
    const float inverse = inverse_scale(min(scale, 253u));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inverse;
    return scale == 255u ? 0u : encode8(v);
}

} // namespace nkb
