// Conversions to and from microscaled 4-bit floats, and the re-ordering of row-major codes into the tile form the tensor
// cores read (nkb_mx.h).
//
// For 32 consecutive values of a row with largest magnitude t the scale is 2^X, X = clamp(floor(log2 t) - 2, -127, 127), so
// that t / 2^X lies in [4, 8) and the largest code is used (values above 6 become 6); each value over the scale is rounded to
// nearest, ties to the even code. X comes from the exponent field of t alone and the division is a multiplication with a
// power of two, so nothing before the one rounding is inexact. A block that holds an infinity or a NaN gets the NaN scale and
// zero codes.
//
// All three kernels are bound by memory: 2 (4) bytes in and 0.53 bytes out per bf16 (f32) value, or the other way round.
#include <cuda_bf16.h>
#include "nkb_decode.cuh"
#include "nkb_mx.h"
#include "nkb_ptx.cuh"

namespace nkb {

namespace {

constexpr int kThreads = 256;

// Where a row's codes and scales go.
struct RowMajorSink {
    uint8_t *codes, *scales;
    uint64_t codes_stride, scales_stride;
};

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

// Eight consecutive values of a row, zeros past `count`. `aligned`: all eight exist and lie on a 16-byte boundary.
template <uint32_t kType>
__device__ __forceinline__ void load8(const uint8_t *p, int count, bool aligned, float (&v)[8]) {
    constexpr int kBytes = kType == kF32 ? 4 : 2;
    if (aligned) {
        if constexpr (kType == kF32) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = decode_bits<kType>(w[i] & 0xffffu); v[2 * i + 1] = decode_bits<kType>(w[i] >> 16); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < count ? decode<kType>(p + i * kBytes) : 0.0f;
    }
}

// One warp turns 256 values of one row (a chunk row) into 128 bytes of codes and 8 scales; a thread has 8 of the values, four
// threads a block. Warps walk the (row, depth block) grid.
template <uint32_t kType, bool kTiled>
__global__ void __launch_bounds__(kThreads) quantise_kernel(const uint8_t *x, uint64_t rows, uint64_t depth, uint64_t x_stride, RowMajorSink out,
                                                            uint8_t *chunks, uint32_t depth_blocks, const int32_t *row_dest, const int32_t *tile_count,
                                                            uint32_t divide) {
    if constexpr (kTiled) allow_next_kernel();  // the product that reads the chunks may set itself up meanwhile
    if (kTiled && row_dest) rows = (uint64_t)*tile_count * kChunkRows;
    constexpr int kBytes = kType == kF32 ? 4 : 2;
    const int lane = threadIdx.x & 31;
    const bool base_aligned = ((reinterpret_cast<uintptr_t>(x) | x_stride) & 15u) == 0;
    const uint64_t items = rows * depth_blocks, step = (uint64_t)gridDim.x * (kThreads / 32);
    for (uint64_t item = (uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += step) {
        const uint64_t row = item / depth_blocks;
        const uint32_t kb = (uint32_t)(item - row * depth_blocks);
        uint64_t from = row;
        if (kTiled && row_dest) {
            const int32_t d = __ldg(row_dest + row);
            if (d < 0) continue;
            from = (uint32_t)d / divide;
        }
        const uint64_t first = (uint64_t)kb * kMxChunkValues + lane * 8;
        const int64_t left = (int64_t)depth - (int64_t)first;
        const int count = left >= 8 ? 8 : left > 0 ? (int)left : 0;
        float v[8];
        load8<kType>(x + from * x_stride + first * kBytes, count, base_aligned && count == 8, v);
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = max(largest, __float_as_uint(v[i]) & 0x7fffffffu);
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const uint32_t s = scale_byte(largest);
        const float inverse = s == 255u ? 0.0f : inverse_scale(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = s == 255u ? 0.0f : v[i] * inverse;
        const uint32_t codes = encode8(v);
        if constexpr (kTiled) {
            uint8_t *chunk = chunks + ((row / kChunkRows) * depth_blocks + kb) * kMxChunkBytes;
            const uint32_t r = (uint32_t)(row % kChunkRows);
            *reinterpret_cast<uint32_t *>(chunk + r * 128u + ((((uint32_t)lane >> 2) ^ (r & 7u)) << 4) + (lane & 3) * 4) = codes;
            if ((lane & 3) == 0)
                chunk[kMxCodeBytes + (lane >> 4) * 512 + (r & 31u) * 16 + (r >> 5) * 4 + ((lane >> 2) & 3)] = (uint8_t)s;
        } else {
            const uint64_t byte = first / 2, row_bytes = (depth + 1) / 2;
            uint8_t *c = out.codes + row * out.codes_stride + byte;
            if (count == 8 && (reinterpret_cast<uintptr_t>(c) & 3u) == 0) *reinterpret_cast<uint32_t *>(c) = codes;
            else
                for (int i = 0; i < 4; ++i)
                    if (byte + i < row_bytes) c[i] = (uint8_t)(codes >> (8 * i));
            if ((lane & 3) == 0 && first < depth) out.scales[row * out.scales_stride + first / kMxBlock] = (uint8_t)s;
        }
    }
}

__device__ __forceinline__ float code_value(uint32_t code) {
    const uint32_t e = (code >> 1) & 3u, m = code & 1u;
    const float size = e == 0 ? 0.5f * m : __uint_as_float(((126u + e) << 23) | (m << 22));
    return code & 8u ? -size : size;
}
__device__ __forceinline__ float scale_value(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7fc00000u) : s == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
}

// Eight codes per thread, written as the values they stand for (rounded to nearest where the type is narrower: f16 only,
// whose range the scale can leave).
template <uint32_t kType>
__global__ void __launch_bounds__(kThreads) dequantise_kernel(const uint8_t *codes, uint64_t codes_stride, const uint8_t *scales, uint64_t scales_stride,
                                                              uint64_t rows, uint64_t depth, uint8_t *x, uint64_t x_stride) {
    constexpr int kBytes = kType == kF32 ? 4 : 2;
    const uint64_t pieces = (depth + 7) / 8, items = rows * pieces, step = (uint64_t)gridDim.x * kThreads;
    for (uint64_t item = (uint64_t)blockIdx.x * kThreads + threadIdx.x; item < items; item += step) {
        const uint64_t row = item / pieces, first = (item - row * pieces) * 8;
        const uint8_t *c = codes + row * codes_stride + first / 2;
        const int count = depth - first >= 8 ? 8 : (int)(depth - first);
        uint32_t w = 0;
        if (count == 8 && (reinterpret_cast<uintptr_t>(c) & 3u) == 0) w = __ldg(reinterpret_cast<const uint32_t *>(c));
        else
            for (int i = 0; i < (count + 1) / 2; ++i) w |= (uint32_t)c[i] << (8 * i);
        const float scale = scale_value(scales[row * scales_stride + first / kMxBlock]);
        uint8_t *dst = x + row * x_stride + first * kBytes;
        const bool whole = count == 8 && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0;
        uint32_t out[kBytes == 4 ? 8 : 4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = code_value((w >> (4 * i)) & 15u) * scale;
            if constexpr (kType == kF32) out[i] = __float_as_uint(v);
            else {
                const uint32_t b = kType == kBF16 ? (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)) : (uint32_t)__half_as_ushort(__float2half_rn(v));
                out[i / 2] = i & 1 ? out[i / 2] | (b << 16) : b;
            }
        }
        if (whole) {
            reinterpret_cast<uint4 *>(dst)[0] = make_uint4(out[0], out[1], out[2], out[3]);
            if constexpr (kType == kF32) reinterpret_cast<uint4 *>(dst)[1] = make_uint4(out[4], out[5], out[6], out[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i >= count) break;
                if constexpr (kType == kF32) memcpy(dst + 4 * i, &out[i], 4);
                else {
                    dst[2 * i] = (uint8_t)(out[i / 2] >> (16 * (i & 1)));
                    dst[2 * i + 1] = (uint8_t)(out[i / 2] >> (16 * (i & 1) + 8));
                }
            }
        }
    }
}

// Row-major codes and scales -> chunks: one warp per chunk row, four bytes of codes per thread. Both codes of the last byte of
// an odd depth count, as for the other 4-bit types; what lies past the depth is zero codes under scale 1.
__global__ void __launch_bounds__(kThreads) tile_kernel(const uint8_t *codes, uint64_t codes_stride, const uint8_t *scales, uint64_t scales_stride,
                                                        uint64_t width, uint64_t depth, uint64_t tiled_rows, uint32_t group_rows, uint8_t *chunks,
                                                        uint32_t depth_blocks) {
    allow_next_kernel();
    const int lane = threadIdx.x & 31;
    const uint64_t row_bytes = (depth + 1) / 2, row_scales = (depth + kMxBlock - 1) / kMxBlock;
    const uint64_t items = tiled_rows * depth_blocks, step = (uint64_t)gridDim.x * (kThreads / 32);
    for (uint64_t item = (uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += step) {
        const uint64_t row = item / depth_blocks;
        const uint32_t kb = (uint32_t)(item - row * depth_blocks);
        const uint64_t group = row / group_rows, in_group = row - group * group_rows;
        const bool real = in_group < width;
        const uint64_t from = group * width + in_group;
        const uint64_t byte = (uint64_t)kb * 128u + lane * 4;
        uint32_t w = 0;
        if (real) {
            const uint8_t *c = codes + from * codes_stride + byte;
            if (byte + 4 <= row_bytes && (reinterpret_cast<uintptr_t>(c) & 3u) == 0) w = __ldg(reinterpret_cast<const uint32_t *>(c));
            else
                for (int i = 0; i < 4; ++i)
                    if (byte + i < row_bytes) w |= (uint32_t)c[i] << (8 * i);
        }
        uint8_t *chunk = chunks + ((row / kChunkRows) * depth_blocks + kb) * kMxChunkBytes;
        const uint32_t r = (uint32_t)(row % kChunkRows);
        *reinterpret_cast<uint32_t *>(chunk + r * 128u + ((((uint32_t)lane >> 2) ^ (r & 7u)) << 4) + (lane & 3) * 4) = w;
        if (lane < 8) {
            const uint64_t block = (uint64_t)kb * 8u + lane;
            const uint8_t s = real && block < row_scales ? scales[from * scales_stride + block] : (uint8_t)127;
            chunk[kMxCodeBytes + (lane >> 2) * 512 + (r & 31u) * 16 + (r >> 5) * 4 + (lane & 3)] = s;
        }
    }
}

// Scale tiles alone: one thread per 16-byte line, i.e. four scales of the rows r, r + 32, r + 64 and r + 96 of a chunk. The
// threads of a warp walk the words of one row, so that the reads are whole lines.
__global__ void __launch_bounds__(kThreads) tile_scales_kernel(const uint8_t *scales, uint64_t scales_stride, uint64_t rows, uint64_t depth,
                                                               uint64_t row_blocks, uint32_t words, uint8_t *tiles) {
    allow_next_kernel();
    const uint64_t row_scales = (depth + kMxBlock - 1) / kMxBlock, items = row_blocks * 32 * words;
    const bool aligned = ((reinterpret_cast<uintptr_t>(scales) | scales_stride) & 3u) == 0;
    for (uint64_t item = (uint64_t)blockIdx.x * kThreads + threadIdx.x; item < items; item += (uint64_t)gridDim.x * kThreads) {
        const uint64_t line = item / words;
        const uint32_t word = (uint32_t)(item - line * words), r = (uint32_t)(line & 31u);
        const uint64_t block = line >> 5, first = (uint64_t)word * 4;
        uint32_t w[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint64_t row = block * kChunkRows + g * 32 + r;
            w[g] = 0x7f7f7f7fu;
            if (row < rows) {
                const uint8_t *s = scales + row * scales_stride + first;
                if (aligned && first + 4 <= row_scales) w[g] = __ldg(reinterpret_cast<const uint32_t *>(s));
                else
                    for (int i = 0; i < 4; ++i)
                        if (first + i < row_scales) w[g] = (w[g] & ~(255u << (8 * i))) | ((uint32_t)s[i] << (8 * i));
            }
        }
        *reinterpret_cast<uint4 *>(tiles + (block * (words / 2) + word / 2) * kMxScaleBytes + (word & 1u) * 512 + r * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

uint32_t grid_for(uint64_t warps) {
    const uint64_t blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
    return (uint32_t)(blocks < 148ull * 8 * 4 ? (blocks ? blocks : 1) : 148ull * 8 * 4);
}

} // namespace

cudaError_t launch_mx_quantise(uint32_t type, const void *x, uint64_t rows, uint64_t depth, uint64_t x_stride, void *codes,
                               uint64_t codes_stride, void *scales, uint64_t scales_stride, cudaStream_t stream) {
    const uint32_t kblocks = (uint32_t)((depth + kMxChunkValues - 1) / kMxChunkValues);
    const RowMajorSink out{static_cast<uint8_t *>(codes), static_cast<uint8_t *>(scales), codes_stride, scales_stride};
    const uint32_t grid = grid_for(rows * kblocks);
    const uint8_t *src = static_cast<const uint8_t *>(x);
    switch (type) {
    case kF32: quantise_kernel<kF32, false><<<grid, kThreads, 0, stream>>>(src, rows, depth, x_stride, out, nullptr, kblocks, nullptr, nullptr, 1); break;
    case kBF16: quantise_kernel<kBF16, false><<<grid, kThreads, 0, stream>>>(src, rows, depth, x_stride, out, nullptr, kblocks, nullptr, nullptr, 1); break;
    case kF16: quantise_kernel<kF16, false><<<grid, kThreads, 0, stream>>>(src, rows, depth, x_stride, out, nullptr, kblocks, nullptr, nullptr, 1); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_mx_quantise_tiled(uint32_t type, const void *x, uint64_t depth, uint64_t x_stride, uint64_t tiled_rows,
                                     const int32_t *row_dest, const int32_t *tile_count, uint32_t divide, void *chunks, cudaStream_t stream) {
    const uint32_t kblocks = (uint32_t)((depth + kMxChunkValues - 1) / kMxChunkValues);
    const RowMajorSink none{nullptr, nullptr, 0, 0};
    const uint32_t grid = grid_for(tiled_rows * kblocks);
    const uint8_t *src = static_cast<const uint8_t *>(x);
    uint8_t *dst = static_cast<uint8_t *>(chunks);
    switch (type) {
    case kF32: quantise_kernel<kF32, true><<<grid, kThreads, 0, stream>>>(src, tiled_rows, depth, x_stride, none, dst, kblocks, row_dest, tile_count, divide); break;
    case kBF16: quantise_kernel<kBF16, true><<<grid, kThreads, 0, stream>>>(src, tiled_rows, depth, x_stride, none, dst, kblocks, row_dest, tile_count, divide); break;
    case kF16: quantise_kernel<kF16, true><<<grid, kThreads, 0, stream>>>(src, tiled_rows, depth, x_stride, none, dst, kblocks, row_dest, tile_count, divide); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_mx_dequantise(uint32_t type, const void *codes, uint64_t codes_stride, const void *scales, uint64_t scales_stride,
                                 uint64_t rows, uint64_t depth, void *x, uint64_t x_stride, cudaStream_t stream) {
    const uint32_t grid = grid_for((rows * ((depth + 7) / 8) + 31) / 32);
    const uint8_t *c = static_cast<const uint8_t *>(codes), *s = static_cast<const uint8_t *>(scales);
    uint8_t *dst = static_cast<uint8_t *>(x);
    switch (type) {
    case kF32: dequantise_kernel<kF32><<<grid, kThreads, 0, stream>>>(c, codes_stride, s, scales_stride, rows, depth, dst, x_stride); break;
    case kBF16: dequantise_kernel<kBF16><<<grid, kThreads, 0, stream>>>(c, codes_stride, s, scales_stride, rows, depth, dst, x_stride); break;
    case kF16: dequantise_kernel<kF16><<<grid, kThreads, 0, stream>>>(c, codes_stride, s, scales_stride, rows, depth, dst, x_stride); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_mx_tile_scales(const void *scales, uint64_t scales_stride, uint64_t rows, uint64_t depth, void *tiles, cudaStream_t stream) {
    const uint64_t row_blocks = (rows + kChunkRows - 1) / kChunkRows;
    const uint32_t words = (uint32_t)((depth + kMxChunkValues - 1) / kMxChunkValues) * 2;
    tile_scales_kernel<<<grid_for(row_blocks * words), kThreads, 0, stream>>>(static_cast<const uint8_t *>(scales), scales_stride, rows, depth, row_blocks, words,
                                                                              static_cast<uint8_t *>(tiles));
    return cudaGetLastError();
}

cudaError_t launch_mx_tile(const void *codes, uint64_t codes_stride, const void *scales, uint64_t scales_stride, uint64_t groups,
                           uint64_t width, uint64_t depth, bool pad_rows, void *chunks, cudaStream_t stream) {
    const uint32_t kblocks = (uint32_t)((depth + kMxChunkValues - 1) / kMxChunkValues);
    const uint64_t group_rows = (width + kChunkRows - 1) / kChunkRows * kChunkRows;
    const uint64_t rows = pad_rows ? groups * group_rows : (groups - 1) * group_rows + width;
    tile_kernel<<<grid_for(rows * kblocks), kThreads, 0, stream>>>(static_cast<const uint8_t *>(codes), codes_stride, static_cast<const uint8_t *>(scales),
                                                                   scales_stride, width, depth, rows, (uint32_t)group_rows,
                                                                   static_cast<uint8_t *>(chunks), kblocks);
    return cudaGetLastError();
}

} // namespace nkb
