// What surrounds the grouped product of the experts: the order of the slots by expert, zero rows for slots without one, and
// the weighted sum of a token's rows.
//
// A slot is one (token, choice) pair. The product wants every expert's slots in row tiles of up to 128, so the slots are
// counted per expert, each expert gets ceil(count / 128) tiles, and each slot a place in its expert's tiles. Which place does
// not matter to the result: rows of a product do not depend on one another.
#include <cuda_bf16.h>
#include "nkb_mx.h"

namespace nkb {

namespace {

constexpr int kOrderThreads = 1024;

__global__ void __launch_bounds__(kOrderThreads) expert_order_kernel(const int32_t *ids, uint32_t slots, uint32_t experts, MxRowTile *tiles,
                                                                     int32_t *tile_count, int32_t *row_dest) {
    __shared__ uint32_t count[kRouteMaxExperts], first_tile[kRouteMaxExperts + 1], taken[kRouteMaxExperts];
    for (uint32_t e = threadIdx.x; e < experts; e += kOrderThreads) { count[e] = 0; taken[e] = 0; }
    __syncthreads();
    for (uint32_t s = threadIdx.x; s < slots; s += kOrderThreads) {
        const int32_t e = ids[s];
        if (e >= 0 && e < (int32_t)experts) atomicAdd(&count[e], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t next = 0;
        for (uint32_t e = 0; e < experts; ++e) { first_tile[e] = next; next += (count[e] + 127u) / 128u; }
        first_tile[experts] = next;
        *tile_count = (int32_t)next;
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += kOrderThreads)
        for (uint32_t t = first_tile[e], left = count[e]; t < first_tile[e + 1]; ++t, left -= 128u) {
            tiles[t].group = (int32_t)e;
            tiles[t].rows = (int32_t)min(left, 128u);
        }
    for (uint32_t i = threadIdx.x; i < first_tile[experts] * 128u; i += kOrderThreads) row_dest[i] = -1;
    __syncthreads();
    for (uint32_t s = threadIdx.x; s < slots; s += kOrderThreads) {
        const int32_t e = ids[s];
        if (e >= 0 && e < (int32_t)experts) row_dest[first_tile[e] * 128u + atomicAdd(&taken[e], 1u)] = (int32_t)s;
    }
}

__global__ void __launch_bounds__(256) zero_unrouted_kernel(const int32_t *ids, uint64_t slots, uint32_t experts, uint8_t *out, uint64_t row_bytes, uint64_t out_stride) {
    for (uint64_t s = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); s < slots; s += (uint64_t)gridDim.x * 8) {
        const int32_t e = ids[s];
        if (e >= 0 && e < (int32_t)experts) continue;
        uint16_t *row = reinterpret_cast<uint16_t *>(out + s * out_stride);  // cells are two or four bytes
        for (uint64_t i = threadIdx.x & 31; i < row_bytes / 2; i += 32) row[i] = 0;
    }
}

template <bool kBf16>
__global__ void __launch_bounds__(256) combine_kernel(const float *y, const float *weights, const int32_t *ids, uint64_t tokens, uint32_t top, uint32_t experts,
                                                      uint64_t width, uint8_t *out, uint64_t out_stride) {
    const uint64_t items = tokens * width;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (uint64_t)gridDim.x * 256) {
        const uint64_t t = i / width, c = i - t * width;
        float sum = 0.0f;
        for (uint32_t j = 0; j < top; ++j) {
            const int32_t e = ids[t * top + j];
            if (e >= 0 && e < (int32_t)experts) sum = fmaf(weights[t * top + j], y[(t * top + j) * width + c], sum);
        }
        if constexpr (kBf16) reinterpret_cast<__nv_bfloat16 *>(out + t * out_stride)[c] = __float2bfloat16_rn(sum);
        else reinterpret_cast<float *>(out + t * out_stride)[c] = sum;
    }
}

uint32_t blocks_for(uint64_t n) { return (uint32_t)(n < 148ull * 32 ? (n ? n : 1) : 148ull * 32); }

} // namespace

cudaError_t launch_expert_order(const int32_t *ids, uint64_t slots, uint32_t experts, MxRowTile *tiles, int32_t *tile_count, int32_t *row_dest,
                                uint64_t max_tiles, cudaStream_t stream) {
    if (slots > 0x7fffff00ull || max_tiles > 0x00ffffffull) return cudaErrorInvalidValue;
    expert_order_kernel<<<1, kOrderThreads, 0, stream>>>(ids, (uint32_t)slots, experts, tiles, tile_count, row_dest);
    return cudaGetLastError();
}

cudaError_t launch_zero_unrouted(const int32_t *ids, uint64_t slots, uint32_t experts, void *out, uint64_t row_bytes, uint64_t out_stride, cudaStream_t stream) {
    zero_unrouted_kernel<<<blocks_for((slots + 7) / 8), 256, 0, stream>>>(ids, slots, experts, static_cast<uint8_t *>(out), row_bytes, out_stride);
    return cudaGetLastError();
}

cudaError_t launch_combine(const float *y, const float *weights, const int32_t *ids, uint64_t tokens, uint32_t top, uint32_t experts, uint64_t width,
                           void *out, bool bf16, uint64_t out_stride, cudaStream_t stream) {
    const uint32_t grid = blocks_for((tokens * width + 255) / 256);
    uint8_t *dst = static_cast<uint8_t *>(out);
    if (bf16) combine_kernel<true><<<grid, 256, 0, stream>>>(y, weights, ids, tokens, top, experts, width, dst, out_stride);
    else combine_kernel<false><<<grid, 256, 0, stream>>>(y, weights, ids, tokens, top, experts, width, dst, out_stride);
    return cudaGetLastError();
}

} // namespace nkb
