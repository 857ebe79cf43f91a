// What surrounds the grouped product of the experts: the order of the slots by expert, zero rows for slots without one, and
// the weighted sum of a token's rows.
//
// A slot is one (token, choice) pair. The product wants every expert's slots in row tiles of up to 128 (or 256), so the slots are
// counted per expert, each expert gets the tiles its count fills, and each slot a place in its expert's tiles. Which place does
// not matter to the result: rows of a product do not depend on one another.
#include <cuda_bf16.h>
#include "nkb_mx.h"
#include "nkb_ptx.cuh"

namespace nkb {

namespace {

constexpr int kOrderThreads = 1024;

// Calls `take(slot, expert)` for every slot in [first, end) that has an expert. Sixteen ids are on their way at a time.
template <class Take>
__device__ __forceinline__ void each_slot(const int32_t *ids, uint32_t first, uint32_t end, uint32_t experts, Take take) {
    constexpr uint32_t kAhead = 16;
    for (uint32_t s0 = first + threadIdx.x; s0 < end; s0 += kAhead * kOrderThreads) {
        int32_t e[kAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) e[i] = end - s0 > i * kOrderThreads ? ids[s0 + i * kOrderThreads] : -1;
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
            if ((uint32_t)e[i] < experts) take(s0 + i * kOrderThreads, (uint32_t)e[i]);  // none below 0 either
    }
}

// A cluster of eight blocks, each with an eighth of the slots: it counts them per expert in its shared memory, reads the others' counts from
// theirs, scans the experts for their tiles and hands out places to its own slots behind those of the blocks before it. What took the time
// in one block was the additions to few counters and the scattered four bytes per slot: 16,384 slots of 32 experts 10.7 us, 7.6 us so.
// (At most 256 slots are ordered where their rows are quantised.)
constexpr uint32_t kOrderBlocks = 8;
__global__ void __cluster_dims__(kOrderBlocks, 1, 1) __launch_bounds__(kOrderThreads)
expert_order_kernel(const int32_t *ids, uint32_t slots, uint32_t experts, MxRowTile *tiles, int32_t *tile_count, int32_t *row_dest, uint32_t tile_rows) {
    static_assert(kRouteMaxExperts <= kOrderThreads, "one thread per expert");
    __shared__ uint32_t count[kRouteMaxExperts], all[kRouteMaxExperts], first_row[kRouteMaxExperts], next_row[kRouteMaxExperts], warp_sums[kOrderThreads / 32];
    const uint32_t t = threadIdx.x, lane = t & 31u, rank = cluster_ctarank();
    const uint32_t share = (slots + kOrderBlocks - 1) / kOrderBlocks, first = min(rank * share, slots), end = min(first + share, slots);
    if (t < experts) count[t] = 0;
    __syncthreads();
    each_slot(ids, first, end, experts, [&](uint32_t, uint32_t e) { atomicAdd(&count[e], 1u); });
    __syncwarp();
    cluster_sync_all();
    uint32_t mine = 0, before = 0;
    if (t < experts)
#pragma unroll
        for (uint32_t b = 0; b < kOrderBlocks; ++b) {
            const uint32_t n = ld_shared_cluster(map_to_cta(smem_u32(&count[t]), b));
            before += b < rank ? n : 0u;
            mine += n;
        }
    const uint32_t my_tiles = (mine + tile_rows - 1u) / tile_rows;
    uint32_t through = my_tiles;  // inclusive sum over the experts
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, through, o);
        if ((int)lane >= o) through += v;
    }
    if (lane == 31u) warp_sums[t >> 5] = through;
    __syncthreads();
    if (t < 32) {
        uint32_t w = warp_sums[t];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, w, o);
            if ((int)lane >= o) w += v;
        }
        warp_sums[t] = w;
    }
    __syncthreads();
    if (t >= 32) through += warp_sums[(t >> 5) - 1];
    if (t == kOrderThreads - 1 && rank == 0) *tile_count = (int32_t)through;
    if (t < experts) {
        uint32_t tile = through - my_tiles, left = mine;
        all[t] = mine;
        first_row[t] = tile * tile_rows;
        next_row[t] = tile * tile_rows + before;
        if (t % kOrderBlocks == rank)
            for (; tile < through; ++tile, left -= tile_rows) tiles[tile] = {(int32_t)t, (int32_t)min(left, tile_rows)};
    }
    __syncwarp();
    cluster_sync_all();  // the others have read this block's counts: it may leave
    each_slot(ids, first, end, experts, [&](uint32_t s, uint32_t e) { row_dest[atomicAdd(&next_row[e], 1u)] = (int32_t)s; });
    // Rows behind an expert's last slot belong to nobody.
    for (uint32_t e = rank + (t >> 5) * kOrderBlocks; e < experts; e += kOrderThreads / 32 * kOrderBlocks)
        for (uint32_t r = all[e] + lane; r < (all[e] + tile_rows - 1u) / tile_rows * tile_rows; r += 32) row_dest[first_row[e] + r] = -1;
}

__global__ void __launch_bounds__(256) zero_unrouted_kernel(const int32_t *ids, uint64_t slots, uint32_t experts, uint8_t *out, uint64_t row_bytes, uint64_t out_stride) {
    for (uint64_t s = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); s < slots; s += (uint64_t)gridDim.x * 8) {
        const int32_t e = ids[s];
        if (e >= 0 && e < (int32_t)experts) continue;
        uint16_t *row = reinterpret_cast<uint16_t *>(out + s * out_stride);  // cells are two or four bytes
        for (uint64_t i = threadIdx.x & 31; i < row_bytes / 2; i += 32) row[i] = 0;
    }
}

// One block per token and stretch of columns: the token's ids and weights are the same for all its threads, and four columns a
// thread keep `top` loads of 16 bytes in flight. Bound by memory: y is read once and the sums are written; 4,096 tokens of four rows
// of 2,048 take 25 us, 168 MB at 6.6 TB/s. Starting it early, as the dependent of the product, slowed the product down by more.
template <bool kBf16>
__global__ void __launch_bounds__(256) combine_kernel(const float *y, const float *weights, const int32_t *ids, uint32_t top, uint32_t experts,
                                                      uint64_t width, uint8_t *out, uint64_t out_stride, bool vectors) {
    const uint64_t t = blockIdx.x;
    const float *rows = y + t * top * width;
    const float *w = weights + t * top;
    const int32_t *id = ids + t * top;
    if (vectors) {
        for (uint64_t c = ((uint64_t)blockIdx.y * 256 + threadIdx.x) * 4; c < width; c += (uint64_t)gridDim.y * 1024) {
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (uint32_t j = 0; j < top; ++j) {
                if ((uint32_t)id[j] >= experts) continue;  // none below 0 either
                const float4 v = __ldcs(reinterpret_cast<const float4 *>(rows + j * width + c));
                const float f = w[j];
                sum = make_float4(fmaf(f, v.x, sum.x), fmaf(f, v.y, sum.y), fmaf(f, v.z, sum.z), fmaf(f, v.w, sum.w));
            }
            if constexpr (kBf16) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
                *reinterpret_cast<uint2 *>(out + t * out_stride + c * 2) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
            } else {
                *reinterpret_cast<float4 *>(out + t * out_stride + c * 4) = sum;
            }
        }
    } else {
        for (uint64_t c = (uint64_t)blockIdx.y * 256 + threadIdx.x; c < width; c += (uint64_t)gridDim.y * 256) {
            float sum = 0.0f;
            for (uint32_t j = 0; j < top; ++j)
                if ((uint32_t)id[j] < experts) sum = fmaf(w[j], rows[j * width + c], sum);
            if constexpr (kBf16) reinterpret_cast<__nv_bfloat16 *>(out + t * out_stride)[c] = __float2bfloat16_rn(sum);
            else reinterpret_cast<float *>(out + t * out_stride)[c] = sum;
        }
    }
}

uint32_t blocks_for(uint64_t n) { return (uint32_t)(n < 148ull * 32 ? (n ? n : 1) : 148ull * 32); }

} // namespace

cudaError_t launch_expert_order(const int32_t *ids, uint64_t slots, uint32_t experts, MxRowTile *tiles, int32_t *tile_count, int32_t *row_dest,
                                uint64_t max_tiles, uint32_t tile_rows, cudaStream_t stream) {
    if (slots > 0x7fffff00ull || max_tiles > 0x00ffffffull) return cudaErrorInvalidValue;
    expert_order_kernel<<<kOrderBlocks, kOrderThreads, 0, stream>>>(ids, (uint32_t)slots, experts, tiles, tile_count, row_dest, tile_rows);
    return cudaGetLastError();
}

cudaError_t launch_zero_unrouted(const int32_t *ids, uint64_t slots, uint32_t experts, void *out, uint64_t row_bytes, uint64_t out_stride, cudaStream_t stream) {
    zero_unrouted_kernel<<<blocks_for((slots + 7) / 8), 256, 0, stream>>>(ids, slots, experts, static_cast<uint8_t *>(out), row_bytes, out_stride);
    return cudaGetLastError();
}

cudaError_t launch_combine(const float *y, const float *weights, const int32_t *ids, uint64_t tokens, uint32_t top, uint32_t experts, uint64_t width,
                           void *out, bool bf16, uint64_t out_stride, cudaStream_t stream) {
    uint8_t *dst = static_cast<uint8_t *>(out);
    const bool vectors = width % 4 == 0 && ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out) | (tokens > 1 ? out_stride : 0)) & 15u) == 0;
    const uint64_t stretches = (width + (vectors ? 1023 : 255)) / (vectors ? 1024 : 256);
    const dim3 grid((uint32_t)tokens, (uint32_t)(stretches < 4096 ? stretches : 4096));
    if (bf16) combine_kernel<true><<<grid, 256, 0, stream>>>(y, weights, ids, top, experts, width, dst, out_stride, vectors);
    else combine_kernel<false><<<grid, 256, 0, stream>>>(y, weights, ids, top, experts, width, dst, out_stride, vectors);
    return cudaGetLastError();
}

} // namespace nkb
