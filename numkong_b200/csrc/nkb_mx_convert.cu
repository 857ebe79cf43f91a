// Conversions to and from microscaled 4-bit floats, and the re-ordering of row-major codes into the tile form the tensor
// cores read (nkb_mx.h).
//
// For 32 consecutive values of a row with largest magnitude t the scale is 2^X, X = clamp(floor(log2 t) - 2, -127, 127), so
// that t / 2^X lies in [4, 8) and the largest code is used (values above 6 become 6); each value over the scale is rounded to
// nearest, ties to the even code. X comes from the exponent field of t alone and the division is a multiplication with a
// power of two, so nothing before the one rounding is inexact. A block that holds an infinity or a NaN gets the NaN scale and
// zero codes.
// (nkb_mx_encode.cuh).
//
// All kernels here are bound by memory: 2 (4) bytes in and 0.53 bytes out per bf16 (f32) value, or the other way round.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "nkb_decode.cuh"
#include "nkb_mx.h"
#include "nkb_mx_encode.cuh"
#include "nkb_ptx.cuh"

namespace nkb {

namespace {

constexpr int kThreads = 256;

// Where a row's codes and scales go.
struct RowMajorSink {
    uint8_t *codes, *scales;
    uint64_t codes_stride, scales_stride;
};

constexpr int kAhead = 4;  // chunk rows (256 values) a warp has in flight

// The warp's piece of work: chunk rows kb0 .. kb0 + ahead of one row (kAhead of them, or one where there are few).
struct Piece {
    uint32_t row, kb0;
};
__device__ __forceinline__ Piece piece_of(uint32_t item, uint32_t pieces_per_row, uint32_t ahead) {
    const uint32_t row = item / pieces_per_row;
    return {row, (item - row * pieces_per_row) * ahead};
}

// The warp's 32 words (lane i: bytes 4 i .. 4 i + 3) to `p`, of which `bytes` exist. Off a four-byte boundary the words are
// shifted into place, so that all but the first and the last few bytes still go out as words.
__device__ __forceinline__ void store_words(uint8_t *p, uint32_t w, uint32_t bytes, int lane) {
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 3u;
    uint8_t *base = p - off;
    const uint32_t before = __shfl_up_sync(0xffffffffu, w, 1);
    const uint32_t shifted = off ? __funnelshift_l(before, w, 8 * off) : w;
    const uint32_t first = 4 * lane;  // offset of this lane's word from `base`; the row's bytes are [off, off + bytes)
    const uint32_t end = off + bytes;
    if (first >= off && first + 4 <= end) *reinterpret_cast<uint32_t *>(base + first) = shifted;
    else
        for (uint32_t i = 0; i < 4; ++i)
            if (first + i >= off && first + i < end) base[first + i] = (uint8_t)(shifted >> (8 * i));
    if (lane == 31 && off)  // what the shift pushed past the last word
        for (uint32_t i = 0; i < off; ++i)
            if (128 + i < end) base[128 + i] = (uint8_t)(w >> (32 - 8 * off + 8 * i));
}

// Codes of one chunk row (lane i: eight values) and its scales (`scales`: lane i the scale of block i % 8) to where they belong.
template <bool kTiled>
__device__ __forceinline__ void store_chunk_row(uint32_t codes, uint32_t row, uint32_t kb, uint64_t depth, const RowMajorSink &out, uint8_t *chunks,
                                                uint32_t depth_blocks, int lane) {
    if constexpr (kTiled) {
        uint8_t *chunk = chunks + ((uint64_t)(row / kChunkRows) * depth_blocks + kb) * kMxCodeBytes;
        const uint32_t r = row % kChunkRows;
        *reinterpret_cast<uint32_t *>(chunk + r * 128u + ((((uint32_t)lane >> 2) ^ (r & 7u)) << 4) + (lane & 3) * 4) = codes;
    } else {
        const uint64_t byte = (uint64_t)kb * 128, row_bytes = (depth + 1) / 2;
        store_words(out.codes + row * out.codes_stride + byte, codes, row_bytes - byte < 128 ? (uint32_t)(row_bytes - byte) : 128u, lane);
    }
}

// A warp turns 256 values of a row (a chunk row) into 128 bytes of codes and eight scales at a time, four such pieces in flight.
//   rows on 16-byte boundaries: a thread loads eight consecutive values, four threads share a block
//   otherwise: a thread loads value `lane` of each block, so that a load still covers whole lines, and the values change hands in
//   shared memory
// 8192 x 8192 bf16: 170 MB in 30 us where the copy rate allows 26; with one piece in flight 50 us.
template <uint32_t kType, bool kTiled>
__device__ __forceinline__ void quantise_piece(const uint8_t *row, const Piece &piece, uint64_t depth, bool aligned, const RowMajorSink &out, uint8_t *chunks,
                                               uint8_t *scale_tiles, uint32_t depth_blocks, uint32_t ahead, uint8_t *staging, int lane) {
    constexpr int kBytes = kType == kF32 ? 4 : 2;
    const uint32_t count = min(ahead, depth_blocks - piece.kb0);
    uint32_t my_scale = 0;  // lane i: the scale of block i % 8 of chunk row kb0 + i / 8
    const uint64_t byte0 = (uint64_t)piece.kb0 * 128 + lane * 4;
    uint8_t *to = kTiled ? chunks + ((uint64_t)(piece.row / kChunkRows) * depth_blocks + piece.kb0) * kMxCodeBytes + (piece.row % kChunkRows) * 128u +
                               ((((uint32_t)lane >> 2) ^ (piece.row & 7u)) << 4) + (lane & 3) * 4
                         : out.codes + piece.row * out.codes_stride + byte0;
    if (aligned && ahead == kAhead && (uint64_t)(piece.kb0 + kAhead) * kMxChunkValues <= depth && (kTiled || (out.codes_stride & 3u) == 0 && (reinterpret_cast<uintptr_t>(out.codes) & 3u) == 0)) {
        // Whole pieces on their boundaries: nothing to guard.
        const uint8_t *from8 = row + ((uint64_t)piece.kb0 * kMxChunkValues + lane * 8) * kBytes;
        uint4 raw[kAhead][kBytes / 2];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int h = 0; h < kBytes / 2; ++h) raw[u][h] = __ldg(reinterpret_cast<const uint4 *>(from8 + u * kMxChunkValues * kBytes) + h);
        uint32_t four = 0;  // this thread's block's scales in the four chunk rows
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            float v[8];
            uint32_t s;
            const uint32_t largest = unpack8<kType>(raw[u], v);
            *reinterpret_cast<uint32_t *>(to + u * (kTiled ? kMxCodeBytes : 128u)) = quantise8(v, largest, s);
            four |= s << (8 * u);
        }
        my_scale = (__shfl_sync(0xffffffffu, four, (lane & 7) * 4) >> (lane & 24)) & 255u;
    } else if (aligned) {
        uint4 raw[kAhead][kBytes / 2];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint64_t first = (uint64_t)(piece.kb0 + u) * kMxChunkValues + lane * 8;
#pragma unroll
            for (int h = 0; h < kBytes / 2; ++h) {
                raw[u][h] = make_uint4(0, 0, 0, 0);
                if (u < (int)ahead && first + 8 <= depth) raw[u][h] = __ldg(reinterpret_cast<const uint4 *>(row + first * kBytes) + h);
            }
            if (u < (int)ahead && first < depth && first + 8 > depth) {  // the row ends inside
                uint32_t w[2 * kBytes] = {};
                for (int i = 0; i < (int)(depth - first); ++i) {
                    if constexpr (kType == kF32) w[i] = __ldg(reinterpret_cast<const uint32_t *>(row) + first + i);
                    else w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(row) + first + i) << (16 * (i & 1));
                }
#pragma unroll
                for (int h = 0; h < kBytes / 2; ++h) raw[u][h] = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (u >= (int)count) break;
            float v[8];
            uint32_t s;
            const uint32_t largest = unpack8<kType>(raw[u], v), codes = quantise8(v, largest, s);
            store_chunk_row<kTiled>(codes, piece.row, piece.kb0 + u, depth, out, chunks, depth_blocks, lane);
            const uint32_t mine = __shfl_sync(0xffffffffu, s, (lane & 7) * 4);
            if ((lane >> 3) == u) my_scale = mine;
        }
    } else {
        uint32_t all[kAhead][8];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const uint64_t at = (uint64_t)(piece.kb0 + u) * kMxChunkValues + b * 32 + lane;
                all[u][b] = 0;
                if (u < (int)count && at < depth) {
                    if constexpr (kType == kF32) all[u][b] = __ldg(reinterpret_cast<const uint32_t *>(row) + at);
                    else all[u][b] = __ldg(reinterpret_cast<const uint16_t *>(row) + at);
                }
            }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (u >= (int)count) break;
            __syncwarp();
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                if constexpr (kType == kF32) reinterpret_cast<uint32_t *>(staging)[b * 32 + lane] = all[u][b];
                else reinterpret_cast<uint16_t *>(staging)[b * 32 + lane] = (uint16_t)all[u][b];
            }
            __syncwarp();
            uint4 raw[kBytes / 2];
#pragma unroll
            for (int h = 0; h < kBytes / 2; ++h) raw[h] = reinterpret_cast<const uint4 *>(staging + lane * 8 * kBytes)[h];
            float v[8];
            uint32_t s;
            const uint32_t largest = unpack8<kType>(raw, v), codes = quantise8(v, largest, s);
            store_chunk_row<kTiled>(codes, piece.row, piece.kb0 + u, depth, out, chunks, depth_blocks, lane);
            const uint32_t mine = __shfl_sync(0xffffffffu, s, (lane & 7) * 4);
            if ((lane >> 3) == u) my_scale = mine;
        }
    }
    if constexpr (kTiled) {
        // Four scales to a word of a scale tile, for which eight lanes of a chunk row hold two words.
        uint32_t word = my_scale << (8 * (lane & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 1);
        word |= __shfl_xor_sync(0xffffffffu, word, 2);
        const uint32_t u = (uint32_t)lane >> 3, r = piece.row % kChunkRows;
        if ((lane & 3) == 0 && u < count)
            *reinterpret_cast<uint32_t *>(scale_tiles + ((uint64_t)(piece.row / kChunkRows) * depth_blocks + piece.kb0 + u) * kMxScaleBytes +
                                          ((lane >> 2) & 1) * 512 + (r & 31u) * 16 + (r >> 5) * 4) = word;
    } else {
        const uint64_t block = (uint64_t)piece.kb0 * 8 + lane;
        if (block * kMxBlock < depth && (uint32_t)(lane >> 3) < count) out.scales[piece.row * out.scales_stride + block] = (uint8_t)my_scale;
    }
}

template <uint32_t kType, bool kTiled>
__global__ void __launch_bounds__(kThreads) quantise_kernel(const uint8_t *x, uint32_t rows, uint64_t depth, uint64_t x_stride, RowMajorSink out,
                                                            uint8_t *chunks, uint8_t *scale_tiles, uint32_t depth_blocks, const int32_t *row_dest,
                                                            const int32_t *tile_count, uint32_t tile_rows, uint32_t divide, uint32_t ahead) {
    if constexpr (kTiled) allow_next_kernel();  // the product that reads the chunks may set itself up meanwhile
    const int lane = threadIdx.x & 31;
    const bool aligned = ((reinterpret_cast<uintptr_t>(x) | x_stride) & 15u) == 0;
    __shared__ __align__(16) uint8_t staging_all[kThreads / 32][kMxChunkValues * (kType == kF32 ? 4 : 2)];
    const uint32_t pieces_per_row = (depth_blocks + ahead - 1) / ahead, items = rows * pieces_per_row;
    const uint32_t used = kTiled && row_dest ? (uint32_t)*tile_count * tile_rows : rows;
    for (uint32_t item = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += gridDim.x * (kThreads / 32)) {
        const Piece piece = piece_of(item, pieces_per_row, ahead);
        uint32_t from = piece.row;
        if (kTiled && row_dest) {
            const int32_t d = row_dest[piece.row];  // whether the row is used comes in at the same time
            if (piece.row >= used) break;
            if (d < 0) continue;
            from = (uint32_t)d / divide;
        }
        quantise_piece<kType, kTiled>(x + (uint64_t)from * x_stride, piece, depth, aligned, out, chunks, scale_tiles, depth_blocks, ahead, staging_all[threadIdx.x >> 5], lane);
    }
}

// The slots of a few tokens: their order by expert (see nkb_experts.cu) and the quantising of their rows in one launch. Every block orders
// all slots for itself, one thread each, in the same way: a slot's row is its expert's first and the number of equal ids before it,
// counted warp by warp. 128 slots of 32 experts, products with 4096 x 2048: 29.3 us for the layer, 32 us with the order and the zeroing as
// launches of their own, 31 us against 38 from Python.
struct FewSlots {
    const int32_t *ids;
    uint32_t slots, experts, divide, tile_rows;
    MxRowTile *tiles;
    int32_t *tile_count, *row_dest;
    uint8_t *out;  // rows of slots without an expert are zeroed here, unless it is null
    uint64_t row_bytes, out_stride;
};
template <uint32_t kType>
__global__ void __launch_bounds__(kThreads) order_and_quantise_kernel(const uint8_t *x, uint64_t depth, uint64_t x_stride, FewSlots f, uint8_t *chunks,
                                                                      uint8_t *scale_tiles, uint32_t depth_blocks, uint32_t ahead) {
    constexpr uint32_t kWarps = kThreads / 32, kPer = kRouteMaxExperts / kThreads;  // experts a thread scans
    static_assert(kFewSlots <= kThreads, "a thread per slot");
    allow_next_kernel();
    __shared__ uint32_t count[kRouteMaxExperts], first_row[kRouteMaxExperts], warp_sums[kWarps];
    __shared__ int32_t row_of[kThreads];
    __shared__ __align__(16) uint8_t staging_all[kWarps][kMxChunkValues * (kType == kF32 ? 4 : 2)];
    const uint32_t t = threadIdx.x, warp = t >> 5;
    const int lane = t & 31;
    const int32_t id = t < f.slots ? f.ids[t] : -1;
    const bool routed = (uint32_t)id < f.experts;  // none below 0 either
    for (uint32_t e = t; e < kRouteMaxExperts; e += kThreads) count[e] = 0;
    const uint32_t same = __match_any_sync(0xffffffffu, routed ? id : -1), before = __popc(same & ((1u << lane) - 1u));
    uint32_t place = before;
    __syncthreads();
    for (uint32_t w = 0; w * 32 < f.slots; ++w) {
        if (warp == w) {
            const uint32_t earlier = routed ? count[id] : 0u;
            __syncwarp();
            place += earlier;
            if (routed && before == 0) count[id] = earlier + __popc(same);
        }
        __syncthreads();
    }
    uint32_t tiles_here[kPer], mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) mine += tiles_here[i] = (count[t * kPer + i] + f.tile_rows - 1) / f.tile_rows;
    uint32_t through = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, through, o);
        if (lane >= o) through += v;
    }
    if (lane == 31) warp_sums[warp] = through;
    __syncthreads();
    for (uint32_t w = 0; w < warp; ++w) through += warp_sums[w];
    if (t == kThreads - 1 && blockIdx.x == 0) *f.tile_count = (int32_t)through;
    uint32_t tile = through - mine;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        first_row[t * kPer + i] = tile * f.tile_rows;
        tile += tiles_here[i];
    }
    __syncthreads();
    if (t < f.slots) row_of[t] = routed ? (int32_t)(first_row[id] + place) : -1;
    if (blockIdx.x == 0 && routed) f.row_dest[first_row[id] + place] = (int32_t)t;
    // The experts' tiles, and the rows behind their last slots, which belong to nobody.
    for (uint32_t e = blockIdx.x * kWarps + warp; e < f.experts; e += gridDim.x * kWarps) {
        const uint32_t slots = count[e], row = first_row[e];
        for (uint32_t r = slots + lane; r < (slots + f.tile_rows - 1) / f.tile_rows * f.tile_rows; r += 32) f.row_dest[row + r] = -1;
        for (uint32_t i = lane; i * f.tile_rows < slots; i += 32) f.tiles[row / f.tile_rows + i] = {(int32_t)e, (int32_t)min(slots - i * f.tile_rows, f.tile_rows)};
    }
    __syncthreads();
    const bool aligned = ((reinterpret_cast<uintptr_t>(x) | x_stride) & 15u) == 0;
    const uint32_t pieces_per_row = (depth_blocks + ahead - 1) / ahead, items = f.slots * pieces_per_row;
    for (uint32_t item = blockIdx.x * kWarps + warp; item < items; item += gridDim.x * kWarps) {
        Piece piece = piece_of(item, pieces_per_row, ahead);
        const uint32_t slot = piece.row;
        const int32_t to = row_of[slot];
        if (to >= 0) {
            piece.row = (uint32_t)to;
            quantise_piece<kType, true>(x + (uint64_t)(slot / f.divide) * x_stride, piece, depth, aligned, RowMajorSink{}, chunks, scale_tiles, depth_blocks, ahead,
                                        staging_all[warp], lane);
        } else if (f.out && piece.kb0 == 0) {
            uint16_t *row = reinterpret_cast<uint16_t *>(f.out + slot * f.out_stride);  // cells are two or four bytes
            for (uint64_t i = lane; i < f.row_bytes / 2; i += 32) row[i] = 0;
        }
    }
}

// Two codes of a byte as values.
__device__ __forceinline__ float2 decode2(uint32_t byte) {
    uint32_t two;
    asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(two) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2 *>(&two));
}
__device__ __forceinline__ float scale_value(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7fc00000u) : s == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
}
template <uint32_t kType>
__device__ __forceinline__ uint32_t encode16(float v) {
    return kType == kBF16 ? (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)) : (uint32_t)__half_as_ushort(__float2half_rn(v));
}

// The way back, a warp per piece as above: the values the codes stand for (rounded to nearest where the type is narrower: f16
// only, whose range the scale can leave). Rows off their boundaries are read byte by byte and written value by value, through shared
// memory, so that a warp's accesses lie side by side. 8192 x 8192 to bf16: 170 MB in 29 us where the copy rate allows 26.
template <uint32_t kType>
__global__ void __launch_bounds__(kThreads) dequantise_kernel(const uint8_t *codes, uint64_t codes_stride, const uint8_t *scales, uint64_t scales_stride,
                                                              uint32_t rows, uint64_t depth, uint8_t *x, uint64_t x_stride, uint32_t depth_blocks,
                                                              uint32_t ahead) {
    constexpr int kBytes = kType == kF32 ? 4 : 2;
    const int lane = threadIdx.x & 31;
    const bool aligned = ((reinterpret_cast<uintptr_t>(x) | x_stride) & 15u) == 0 && ((reinterpret_cast<uintptr_t>(codes) | codes_stride) & 3u) == 0;
    __shared__ __align__(16) uint8_t staging_all[kThreads / 32][kMxChunkValues * kBytes];
    uint8_t *staging = staging_all[threadIdx.x >> 5];
    const uint64_t row_bytes = (depth + 1) / 2;
    const uint32_t pieces_per_row = (depth_blocks + ahead - 1) / ahead, items = rows * pieces_per_row;
    for (uint32_t item = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += gridDim.x * (kThreads / 32)) {
        const Piece piece = piece_of(item, pieces_per_row, ahead);
        const uint32_t count = min(ahead, depth_blocks - piece.kb0);
        const uint8_t *row = codes + piece.row * codes_stride;
        uint8_t *to = x + piece.row * x_stride;
        const uint64_t block = (uint64_t)piece.kb0 * 8 + lane;
        const uint32_t my_scale = block * kMxBlock < depth ? scales[piece.row * scales_stride + block] : 0u;
        if (aligned && ahead == kAhead && (uint64_t)(piece.kb0 + kAhead) * kMxChunkValues <= depth) {
            // Whole pieces on their boundaries: nothing to guard.
            const uint8_t *from8 = row + (uint64_t)piece.kb0 * 128 + lane * 4;
            uint8_t *to8 = to + ((uint64_t)piece.kb0 * kMxChunkValues + lane * 8) * kBytes;
            uint32_t w[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) w[u] = __ldg(reinterpret_cast<const uint32_t *>(from8 + u * 128));
            const float own_scale = scale_value(my_scale);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float scale = __shfl_sync(0xffffffffu, own_scale, u * 8 + (lane >> 2));
                uint32_t value[2 * kBytes];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 v = decode2((w[u] >> (8 * i)) & 255u);
                    if constexpr (kType == kF32) {
                        value[2 * i] = __float_as_uint(v.x * scale);
                        value[2 * i + 1] = __float_as_uint(v.y * scale);
                    } else if constexpr (kType == kBF16) {
                        const __nv_bfloat162 two = __floats2bfloat162_rn(v.x * scale, v.y * scale);
                        value[i] = *reinterpret_cast<const uint32_t *>(&two);
                    } else {
                        const __half2 two = __floats2half2_rn(v.x * scale, v.y * scale);
                        value[i] = *reinterpret_cast<const uint32_t *>(&two);
                    }
                }
#pragma unroll
                for (int h = 0; h < kBytes / 2; ++h)
                    reinterpret_cast<uint4 *>(to8 + u * kMxChunkValues * kBytes)[h] = make_uint4(value[4 * h], value[4 * h + 1], value[4 * h + 2], value[4 * h + 3]);
            }
        } else if (aligned) {
            uint32_t w[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const uint64_t byte = (uint64_t)(piece.kb0 + u) * 128 + lane * 4;
                w[u] = 0;
                if (u >= (int)ahead) continue;
                if (byte + 4 <= row_bytes) w[u] = __ldg(reinterpret_cast<const uint32_t *>(row + byte));
                else
                    for (int i = 0; i < 4; ++i)
                        if (byte + i < row_bytes) w[u] |= (uint32_t)row[byte + i] << (8 * i);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (u >= (int)ahead) break;  // the next warps' chunk rows
                const float scale = scale_value(__shfl_sync(0xffffffffu, my_scale, u * 8 + (lane >> 2)));
                const uint64_t first = (uint64_t)(piece.kb0 + u) * kMxChunkValues + lane * 8;
                uint32_t out[2 * kBytes];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 v = decode2((w[u] >> (8 * i)) & 255u);
                    if constexpr (kType == kF32) {
                        out[2 * i] = __float_as_uint(v.x * scale);
                        out[2 * i + 1] = __float_as_uint(v.y * scale);
                    } else {
                        out[i] = encode16<kType>(v.x * scale) | (encode16<kType>(v.y * scale) << 16);
                    }
                }
                if (first + 8 <= depth) {
#pragma unroll
                    for (int h = 0; h < kBytes / 2; ++h)
                        reinterpret_cast<uint4 *>(to + first * kBytes)[h] = make_uint4(out[4 * h], out[4 * h + 1], out[4 * h + 2], out[4 * h + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (first + i >= depth) break;
                        if constexpr (kType == kF32) reinterpret_cast<uint32_t *>(to)[first + i] = out[i];
                        else reinterpret_cast<uint16_t *>(to)[first + i] = (uint16_t)(out[i / 2] >> (16 * (i & 1)));
                    }
                }
            }
        } else {
            uint32_t w[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const uint64_t byte = (uint64_t)(piece.kb0 + u) * 128 + lane * 4;
                w[u] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (u < (int)count && byte + i < row_bytes) w[u] |= (uint32_t)__ldg(row + byte + i) << (8 * i);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (u >= (int)count) break;
                const float scale = scale_value(__shfl_sync(0xffffffffu, my_scale, u * 8 + (lane >> 2)));
                uint32_t value[2 * kBytes];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 v = decode2((w[u] >> (8 * i)) & 255u);
                    if constexpr (kType == kF32) {
                        value[2 * i] = __float_as_uint(v.x * scale);
                        value[2 * i + 1] = __float_as_uint(v.y * scale);
                    } else {
                        value[i] = encode16<kType>(v.x * scale) | (encode16<kType>(v.y * scale) << 16);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int h = 0; h < kBytes / 2; ++h)
                    reinterpret_cast<uint4 *>(staging + lane * 8 * kBytes)[h] = make_uint4(value[4 * h], value[4 * h + 1], value[4 * h + 2], value[4 * h + 3]);
                __syncwarp();
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    const uint64_t at = (uint64_t)(piece.kb0 + u) * kMxChunkValues + b * 32 + lane;
                    if (at < depth) {
                        if constexpr (kType == kF32) reinterpret_cast<uint32_t *>(to)[at] = reinterpret_cast<const uint32_t *>(staging)[b * 32 + lane];
                        else reinterpret_cast<uint16_t *>(to)[at] = reinterpret_cast<const uint16_t *>(staging)[b * 32 + lane];
                    }
                }
            }
        }
    }
}

// Bytes [0, count) from any address, four to a thread: aligned words, of which only those that hold one of the bytes are read, shifted into
// place. `count` may be negative.
__device__ __forceinline__ uint32_t load_words(const uint8_t *p, int64_t count, int lane) {
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 3u;
    const uint32_t *from = reinterpret_cast<const uint32_t *>(p - off);
    const int64_t end = count > 0 ? count + off : 0;
    const uint32_t w = 4 * lane < end ? __ldg(from + lane) : 0u;
    uint32_t behind = __shfl_down_sync(0xffffffffu, w, 1);
    if (lane == 31) behind = off != 0 && 128 < end ? __ldg(from + 32) : 0u;
    const uint32_t v = __funnelshift_r(w, behind, 8 * off);
    const int64_t left = count - 4 * lane;
    return left >= 4 ? v : left > 0 ? v & ((1u << (8 * (int)left)) - 1u) : 0u;
}

// Row-major codes and scales -> chunks: one warp per piece of up to four chunk rows, four bytes of codes per thread. Both codes of the
// last byte of an odd depth count, as for the other 4-bit types; what lies past the depth is zero codes under scale 1.
// 65,536 x 2048: 143 MB in 71 us, a third of the copy rate; a weight is packed once.
__global__ void __launch_bounds__(kThreads) tile_kernel(const uint8_t *codes, uint64_t codes_stride, const uint8_t *scales, uint64_t scales_stride,
                                                        uint32_t width, uint64_t depth, uint32_t tiled_rows, uint32_t group_rows, uint8_t *chunks,
                                                        uint8_t *scale_tiles, uint32_t depth_blocks, uint32_t ahead) {
    allow_next_kernel();
    const int lane = threadIdx.x & 31;
    const uint64_t row_bytes = (depth + 1) / 2, row_scales = (depth + kMxBlock - 1) / kMxBlock;
    const uint32_t pieces_per_row = (depth_blocks + ahead - 1) / ahead, items = tiled_rows * pieces_per_row;
    for (uint32_t item = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += gridDim.x * (kThreads / 32)) {
        const Piece piece = piece_of(item, pieces_per_row, ahead);
        const uint32_t group = piece.row / group_rows, in_group = piece.row - group * group_rows, r = piece.row % kChunkRows;
        const uint32_t count = min(ahead, depth_blocks - piece.kb0);
        const bool real = in_group < width;
        const uint64_t from = (uint64_t)group * width + in_group;
        uint32_t w[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint64_t byte = (uint64_t)(piece.kb0 + u) * 128u;
            w[u] = load_words(codes + from * codes_stride + byte, real && u < (int)count ? (int64_t)row_bytes - (int64_t)byte : 0, lane);
        }
        const uint64_t block = (uint64_t)piece.kb0 * 8u + lane;  // lane i: the scale of block i % 8 of chunk row kb0 + i / 8
        const uint32_t s = real && block < row_scales ? scales[from * scales_stride + block] : 127u;
        const uint64_t at = (uint64_t)(piece.row / kChunkRows) * depth_blocks + piece.kb0;
        uint8_t *chunk = chunks + at * kMxCodeBytes + r * 128u + ((((uint32_t)lane >> 2) ^ (r & 7u)) << 4) + (lane & 3) * 4;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (u < (int)count) *reinterpret_cast<uint32_t *>(chunk + u * kMxCodeBytes) = w[u];
        uint32_t four = s << (8 * (lane & 3));
        four |= __shfl_xor_sync(0xffffffffu, four, 1);
        four |= __shfl_xor_sync(0xffffffffu, four, 2);
        if ((lane & 3) == 0 && (uint32_t)(lane >> 3) < count)
            *reinterpret_cast<uint32_t *>(scale_tiles + (at + (lane >> 3)) * kMxScaleBytes + ((lane >> 2) & 1) * 512 + (r & 31u) * 16 + (r >> 5) * 4) = four;
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

// Chunk rows a warp takes. So few that the GPU has warps to spare go to one warp each; beyond, four in flight a warp make up for fewer of
// them. Rows of 2048 and of 8192 values alike, one against four, to 4 bits / bf16 back in us: 64 chunk rows 1.79 against 1.92 / 1.53 against
// 1.66; 1024 1.95 against 1.98 / 1.67 against 1.75; 2048 2.12 against 1.99 / 1.84 against 1.79; 4096 2.95 against 2.10 / 2.31 against 1.84.
// (Back to f32 one is the faster at every size measured, 65,536 chunk rows 14.1 against 17.6.)
uint32_t ahead_for(uint64_t rows, uint32_t kblocks) { return rows * kblocks < 2048 ? 1 : kAhead; }
uint64_t pieces(uint32_t kblocks, uint32_t ahead) { return (kblocks + ahead - 1) / ahead; }  // per row
uint32_t grid_for(uint64_t warps) {
    const uint64_t blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
    return (uint32_t)(blocks < 148ull * 8 * 4 ? (blocks ? blocks : 1) : 148ull * 8 * 4);
}

} // namespace

cudaError_t launch_mx_quantise(uint32_t type, const void *x, uint64_t rows, uint64_t depth, uint64_t x_stride, void *codes,
                               uint64_t codes_stride, void *scales, uint64_t scales_stride, cudaStream_t stream) {
    const uint32_t kblocks = (uint32_t)((depth + kMxChunkValues - 1) / kMxChunkValues);
    if (rows == 1) x_stride = 0;  // no stride to be aligned
    const RowMajorSink out{static_cast<uint8_t *>(codes), static_cast<uint8_t *>(scales), codes_stride, scales_stride};
    const uint32_t ahead = ahead_for(rows, kblocks);
    if (rows * pieces(kblocks, ahead) > 0xffffffffull - 148ull * 64 * 8) return cudaErrorInvalidValue;
    const uint32_t grid = grid_for(rows * pieces(kblocks, ahead)), n = (uint32_t)rows;
    const uint8_t *src = static_cast<const uint8_t *>(x);
    switch (type) {
    case kF32: quantise_kernel<kF32, false><<<grid, kThreads, 0, stream>>>(src, n, depth, x_stride, out, nullptr, nullptr, kblocks, nullptr, nullptr, 0, 1, ahead); break;
    case kBF16: quantise_kernel<kBF16, false><<<grid, kThreads, 0, stream>>>(src, n, depth, x_stride, out, nullptr, nullptr, kblocks, nullptr, nullptr, 0, 1, ahead); break;
    case kF16: quantise_kernel<kF16, false><<<grid, kThreads, 0, stream>>>(src, n, depth, x_stride, out, nullptr, nullptr, kblocks, nullptr, nullptr, 0, 1, ahead); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_mx_quantise_tiled(uint32_t type, const void *x, uint64_t depth, uint64_t x_stride, uint64_t tiled_rows,
                                     const int32_t *row_dest, const int32_t *tile_count, uint32_t tile_rows, uint32_t divide, void *chunks, cudaStream_t stream) {
    const uint32_t kblocks = (uint32_t)((depth + kMxChunkValues - 1) / kMxChunkValues);
    const RowMajorSink none{nullptr, nullptr, 0, 0};
    const uint32_t ahead = ahead_for(tiled_rows, kblocks);
    if (tiled_rows * pieces(kblocks, ahead) > 0xffffffffull - 148ull * 64 * 8) return cudaErrorInvalidValue;
    // Rows found through row_dest are a latency each: warps that take several of them meet it less often than new blocks do. 16,384 rows of
    // 2,048 bf16 in a layer of experts: 69.3 us with eight blocks per SM, 70.6 with 32.
    uint32_t grid = grid_for(tiled_rows * pieces(kblocks, ahead));
    if (row_dest && grid > 148 * 8) grid = 148 * 8;
    const uint32_t n = (uint32_t)tiled_rows;
    const uint8_t *src = static_cast<const uint8_t *>(x);
    uint8_t *dst = static_cast<uint8_t *>(chunks), *tiles = dst + (tiled_rows + kChunkRows - 1) / kChunkRows * kblocks * kMxCodeBytes;
    switch (type) {
    case kF32: quantise_kernel<kF32, true><<<grid, kThreads, 0, stream>>>(src, n, depth, x_stride, none, dst, tiles, kblocks, row_dest, tile_count, tile_rows, divide, ahead); break;
    case kBF16: quantise_kernel<kBF16, true><<<grid, kThreads, 0, stream>>>(src, n, depth, x_stride, none, dst, tiles, kblocks, row_dest, tile_count, tile_rows, divide, ahead); break;
    case kF16: quantise_kernel<kF16, true><<<grid, kThreads, 0, stream>>>(src, n, depth, x_stride, none, dst, tiles, kblocks, row_dest, tile_count, tile_rows, divide, ahead); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_order_and_quantise(uint32_t type, const void *x, uint64_t depth, uint64_t x_stride, const int32_t *ids, uint32_t slots, uint32_t experts, uint32_t divide,
                                      uint32_t tile_rows, uint64_t max_tiles, MxRowTile *tiles, int32_t *tile_count, int32_t *row_dest, void *out,
                                      uint64_t row_bytes, uint64_t out_stride, void *chunks, cudaStream_t stream) {
    if (slots > kFewSlots || experts > kRouteMaxExperts) return cudaErrorInvalidValue;
    const uint32_t kblocks = (uint32_t)((depth + kMxChunkValues - 1) / kMxChunkValues), ahead = ahead_for(slots, kblocks);
    const uint32_t grid = grid_for(slots * pieces(kblocks, ahead));
    const FewSlots f{ids, slots, experts, divide, tile_rows, tiles, tile_count, row_dest, static_cast<uint8_t *>(out), row_bytes, out_stride};
    const uint8_t *src = static_cast<const uint8_t *>(x);
    uint8_t *dst = static_cast<uint8_t *>(chunks), *scale_tiles = dst + max_tiles * (tile_rows / kChunkRows) * kblocks * kMxCodeBytes;
    switch (type) {
    case kF32: order_and_quantise_kernel<kF32><<<grid, kThreads, 0, stream>>>(src, depth, x_stride, f, dst, scale_tiles, kblocks, ahead); break;
    case kBF16: order_and_quantise_kernel<kBF16><<<grid, kThreads, 0, stream>>>(src, depth, x_stride, f, dst, scale_tiles, kblocks, ahead); break;
    case kF16: order_and_quantise_kernel<kF16><<<grid, kThreads, 0, stream>>>(src, depth, x_stride, f, dst, scale_tiles, kblocks, ahead); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_mx_dequantise(uint32_t type, const void *codes, uint64_t codes_stride, const void *scales, uint64_t scales_stride,
                                 uint64_t rows, uint64_t depth, void *x, uint64_t x_stride, cudaStream_t stream) {
    const uint32_t kblocks = (uint32_t)((depth + kMxChunkValues - 1) / kMxChunkValues);
    const uint32_t ahead = ahead_for(rows, kblocks);
    if (rows * pieces(kblocks, ahead) > 0xffffffffull - 148ull * 64 * 8) return cudaErrorInvalidValue;
    const uint32_t grid = grid_for(rows * pieces(kblocks, ahead)), n = (uint32_t)rows;
    if (rows == 1) codes_stride = x_stride = 0;
    const uint8_t *c = static_cast<const uint8_t *>(codes), *s = static_cast<const uint8_t *>(scales);
    uint8_t *dst = static_cast<uint8_t *>(x);
    switch (type) {
    case kF32: dequantise_kernel<kF32><<<grid, kThreads, 0, stream>>>(c, codes_stride, s, scales_stride, n, depth, dst, x_stride, kblocks, ahead); break;
    case kBF16: dequantise_kernel<kBF16><<<grid, kThreads, 0, stream>>>(c, codes_stride, s, scales_stride, n, depth, dst, x_stride, kblocks, ahead); break;
    case kF16: dequantise_kernel<kF16><<<grid, kThreads, 0, stream>>>(c, codes_stride, s, scales_stride, n, depth, dst, x_stride, kblocks, ahead); break;
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
    const uint32_t ahead = ahead_for(rows, kblocks);
    if (rows * pieces(kblocks, ahead) > 0xffffffffull - 148ull * 64 * 8) return cudaErrorInvalidValue;
    uint8_t *dst = static_cast<uint8_t *>(chunks);
    tile_kernel<<<grid_for(rows * pieces(kblocks, ahead)), kThreads, 0, stream>>>(static_cast<const uint8_t *>(codes), codes_stride, static_cast<const uint8_t *>(scales),
                                                                                  scales_stride, (uint32_t)width, depth, (uint32_t)rows, (uint32_t)group_rows, dst,
                                                                                  dst + groups * group_rows / kChunkRows * kblocks * kMxCodeBytes, kblocks, ahead);
    return cudaGetLastError();
}

} // namespace nkb
