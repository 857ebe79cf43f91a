// Product of two MXFP4 operands in tile form (nkb_mx.h): C = A . B^T with f32 accumulation, f32 or bf16 cells, one packed
// matrix or a group of them.
//
//   C[i, j] = sum over blocks b of 2^(sa[i,b] + sb[j,b] - 254) * sum over the block's 32 values of a_l b_l
//
// tcgen05.mma.kind::mxf4 takes 64 values of depth a step and applies the scales inside: the scales come from TMEM, where
// tcgen05.cp puts the chunk's scale tiles just before the chunk's MMAs (both run in the order one thread issues them).
// e2m1 products are multiples of 1/4 of at most 36, so a block's sum is exact and the accumulator only loses bits when the
// block scales of a row spread over more than 2^10.
//
// One persistent CTA per SM, ten warps, as in the packed GEMM of the other types: warp 0 brings chunks to shared memory with
// untiled bulk copies, warp 1 issues copies of scales and MMAs, warps 2..9 read the accumulators out and store the cells.
#include <cuda_bf16.h>
#include "nkb_mx.h"
#include "nkb_ptx.cuh"

namespace nkb {

namespace {

constexpr int kBM = 128;
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 64 + 32 * kEpilogueWarps;
constexpr int kStepBytes = 32;       // bytes of depth (64 values) one MMA consumes
constexpr uint32_t kGroupM = 8;      // row tiles walked before the next column tile

struct MxGemmDev {
    const uint8_t *a_chunks, *b_chunks;
    uint8_t *c;
    uint64_t c_stride;
    uint32_t m, n, kblocks;
    uint32_t tiles_m, tiles_n;
    uint32_t group_blocks;           // row blocks of 128 per packed matrix
    const MxRowTile *tiles;
    const int32_t *tile_count, *row_dest;
    unsigned int *error_word;
    uint32_t wait_us[kWaitSites];
};

template <int kBN, int kStages>
struct Plan {
    static constexpr int kBBytes = kBN * 128;
    static constexpr int kScaleOffset = kBM * 128 + kBBytes;           // A codes, B codes, A scales, B scales
    static constexpr int kStageBytes = kScaleOffset + kMxScaleBytes + kBN / 128 * kMxScaleBytes;
    static constexpr int kBarrierOffset = kStages * kStageBytes;
    static constexpr int kStagingPitch = 144;                          // bytes per staged row: 128 and one 16-byte piece against bank conflicts
    static constexpr int kStagingOffset = kBarrierOffset + 256;
    static constexpr int kTotal = kStagingOffset + kEpilogueWarps * 32 * kStagingPitch + 1024;
};

__device__ __forceinline__ void tile_coords(uint32_t tile, uint32_t tiles_m, uint32_t tiles_n, uint32_t &mt, uint32_t &nt) {
    const uint32_t per_group = kGroupM * tiles_n, group = tile / per_group, first = group * kGroupM;
    const uint32_t rows = min(tiles_m - first, kGroupM), in_group = tile % per_group;
    mt = first + in_group % rows;
    nt = in_group / rows;
    if (group & 1u) nt = tiles_n - 1u - nt;  // the packed rows touched last are still in L2
}

// Stores this thread's row x kCols f32 accumulators: 128 bytes of a row at a time go through the warp's staging block, so that
// each store instruction writes whole 128-byte lines. `dest` is this lane's destination row, negative for none.
template <bool kBf16, int kCols>
__device__ __forceinline__ void store_rows(const uint32_t (&acc)[kCols], const MxGemmDev &p, int64_t dest, uint32_t col_base, uint8_t *staging, int pitch, int lane) {
    constexpr int kPieceCols = kBf16 ? 64 : 32;  // columns in 128 bytes
    constexpr int kCell = kBf16 ? 2 : 4;
    static_assert(kCols % kPieceCols == 0, "whole pieces");
    if (!__any_sync(0xffffffffu, dest >= 0)) return;
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.c) | p.c_stride) & 15u) == 0;
#pragma unroll
    for (int c = 0; c < kCols / kPieceCols; ++c) {
        const uint32_t col0 = col_base + c * kPieceCols;
        if (col0 >= p.n) break;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            uint4 v;
            if constexpr (kBf16) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 two = __floats2bfloat162_rn(__uint_as_float(acc[c * 64 + q * 8 + 2 * j]), __uint_as_float(acc[c * 64 + q * 8 + 2 * j + 1]));
                    w[j] = *reinterpret_cast<const uint32_t *>(&two);
                }
                v = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                v = make_uint4(acc[c * 32 + q * 4], acc[c * 32 + q * 4 + 1], acc[c * 32 + q * 4 + 2], acc[c * 32 + q * 4 + 3]);
            }
            *reinterpret_cast<uint4 *>(staging + lane * pitch + q * 16) = v;
        }
        __syncwarp();
#pragma unroll
        for (int it = 0; it < 8; ++it) {
            const int r = it * 4 + lane / 8, q = lane % 8;
            const int64_t row = __shfl_sync(0xffffffffu, dest, r);
            const uint32_t col = col0 + q * (16 / kCell);
            if (row >= 0 && col < p.n) {
                const uint4 v = *reinterpret_cast<const uint4 *>(staging + r * pitch + q * 16);
                uint8_t *dst = p.c + (uint64_t)row * p.c_stride + (uint64_t)col * kCell;
                if (aligned && col + 16 / kCell <= p.n) __stcs(reinterpret_cast<uint4 *>(dst), v);
                else {
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 16 / kCell; ++j)
                        if (col + j < p.n) {
                            if constexpr (kBf16) *reinterpret_cast<uint16_t *>(dst + 2 * j) = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
                            else *reinterpret_cast<uint32_t *>(dst + 4 * j) = w[j];
                        }
                }
            }
        }
        __syncwarp();
    }
}

template <int kBN, int kStages, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1) gemm_mx_kernel(const MxGemmDev p) {
    using P = Plan<kBN, kStages>;
    constexpr int kColsPerThread = kBN / 2;
    constexpr int kScaleCols = 8 + kBN / 16;                 // one chunk's scales: two words per row of A and of B
    constexpr int kTmemCols = 512;
    static_assert(2 * kBN + kScaleCols <= kTmemCols, "two accumulators and the scales fit TMEM");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bar_base = smem_base + P::kBarrierOffset;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
    auto tmem_full_bar = [&](int a) { return bar_base + 8u * (2 * kStages + a); };
    auto tmem_empty_bar = [&](int a) { return bar_base + 8u * (2 * kStages + 2 + a); };
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + P::kBarrierOffset + 8 * (2 * kStages + 4));
    const uint32_t drain_bar = bar_base + 8u * (2 * kStages + 5);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(tmem_full_bar(a), 1); mbar_init(tmem_empty_bar(a), kEpilogueWarps * 32); }
        mbar_init(drain_bar, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t *>(tmem_slot)), kTmemCols);
        tmem_relinquish<1>();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tiles_m = p.tile_count ? (uint32_t)*p.tile_count : p.tiles_m;
    const uint32_t num_tiles = tiles_m * p.tiles_n;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0, issued = 0;
            bool ok = true;
            for (uint32_t tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
                uint32_t mt, nt;
                tile_coords(tile, tiles_m, p.tiles_n, mt, nt);
                const uint32_t rows = p.tiles ? (uint32_t)p.tiles[mt].rows : min(p.m - mt * kBM, (uint32_t)kBM);
                const uint32_t group = p.tiles ? (uint32_t)p.tiles[mt].group : 0u;
                // Only the row groups of eight that hold valid rows are fetched; what the rest of the buffer holds ends up in
                // rows of the accumulator that nobody reads.
                const uint32_t a_bytes = (rows + 7u) / 8u * 1024u;
                const uint32_t block0 = nt * (kBN / 128), blocks = min((uint32_t)(kBN / 128), p.group_blocks - block0);
                const uint8_t *a_src = p.a_chunks + (uint64_t)mt * p.kblocks * kMxChunkBytes;
                const uint8_t *b_src = p.b_chunks + ((uint64_t)group * p.group_blocks + block0) * p.kblocks * kMxChunkBytes;
                for (uint32_t kb = 0; kb < p.kblocks; ++kb) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, 1, p.error_word, p.wait_us[1])) { ok = false; break; }
                    const uint32_t dst = smem_base + stage * P::kStageBytes;
                    mbar_expect_tx(full_bar(stage), a_bytes + kMxScaleBytes + blocks * kMxChunkBytes);
                    const uint8_t *a = a_src + (uint64_t)kb * kMxChunkBytes;
                    bulk_load(dst, a, a_bytes, full_bar(stage));
                    bulk_load(dst + P::kScaleOffset, a + kMxCodeBytes, kMxScaleBytes, full_bar(stage));
                    for (uint32_t j = 0; j < blocks; ++j) {
                        const uint8_t *b = b_src + ((uint64_t)j * p.kblocks + kb) * kMxChunkBytes;
                        bulk_load(dst + kBM * 128 + j * kMxCodeBytes, b, kMxCodeBytes, full_bar(stage));
                        bulk_load(dst + P::kScaleOffset + (1 + j) * kMxScaleBytes, b + kMxCodeBytes, kMxScaleBytes, full_bar(stage));
                    }
                    ++issued;
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
            if (!ok) {  // copies in flight must land before the block may retire
                int s = stage;
                uint32_t ph = phase;
                for (uint32_t i = 0; i < issued && i < (uint32_t)kStages; ++i) {
                    if (s == 0) { s = kStages; ph ^= 1u; }
                    --s;
                    if (!mbar_wait(full_bar(s), ph, 6, p.error_word, p.wait_us[6])) break;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0, seq = 0;
            bool ok = true;
            const uint32_t scales_a = tmem_base + 2 * kBN, scales_b = scales_a + 8;
            for (uint32_t tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++seq) {
                const uint32_t buf = seq & 1u, buf_phase = (seq >> 1) & 1u;
                if (!mbar_wait(tmem_empty_bar(buf), buf_phase ^ 1u, 2, p.error_word, p.wait_us[2])) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + buf * kBN;
                for (uint32_t kb = 0; kb < p.kblocks; ++kb) {
                    if (!mbar_wait(full_bar(stage), phase, 3, p.error_word, p.wait_us[3])) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint32_t src = smem_base + stage * P::kStageBytes;
                    const uint64_t a_desc = make_smem_desc_sw128(src), b_desc = make_smem_desc_sw128(src + kBM * 128);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {  // two scale tiles, 128 values of depth each
                        tmem_copy_scales<1>(scales_a + t * 4, make_smem_desc_scales(src + P::kScaleOffset + t * 512));
#pragma unroll
                        for (int j = 0; j < kBN / 128; ++j)
                            tmem_copy_scales<1>(scales_b + t * (kBN / 32) + j * 4, make_smem_desc_scales(src + P::kScaleOffset + (1 + j) * kMxScaleBytes + t * 512));
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_mxf4<1>(d_tmem, a_desc + 2u * k, b_desc + 2u * k, make_idesc_mxf4(kBM, kBN, (k & 1) * 2),
                                     scales_a + (k >> 1) * 4, scales_b + (k >> 1) * (kBN / 32), (kb | (uint32_t)k) != 0u);
                    umma_commit(empty_bar(stage));
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
                if (ok) umma_commit(tmem_full_bar(buf));
            }
            umma_commit(drain_bar);  // shared memory and TMEM are released below: the last MMAs must have retired
            mbar_wait(drain_bar, 0u, 5, p.error_word, p.wait_us[5]);
        }
    } else {
        const uint32_t quarter = warp & 3u, half = (uint32_t)(warp - 2) >> 2;
        uint8_t *staging = smem_gen + P::kStagingOffset + (warp - 2) * 32 * P::kStagingPitch;
        uint32_t seq = 0;
        for (uint32_t tile = blockIdx.x; tile < num_tiles; tile += gridDim.x, ++seq) {
            uint32_t mt, nt;
            tile_coords(tile, tiles_m, p.tiles_n, mt, nt);
            const uint32_t buf = seq & 1u, buf_phase = (seq >> 1) & 1u;
            const uint32_t in_tile = quarter * 32u + lane;
            const uint32_t rows = p.tiles ? (uint32_t)p.tiles[mt].rows : min(p.m - mt * kBM, (uint32_t)kBM);
            int64_t dest = -1;
            if (in_tile < rows) dest = p.row_dest ? (int64_t)p.row_dest[(uint64_t)mt * kBM + in_tile] : (int64_t)mt * kBM + in_tile;
            // The whole warp leaves together: the stores below synchronise it.
            if (!__all_sync(0xffffffffu, mbar_wait(tmem_full_bar(buf), buf_phase, 4, p.error_word, p.wait_us[4]))) break;
            tc_fence_after_sync();
            uint32_t acc[kColsPerThread];
#pragma unroll
            for (int c = 0; c < kColsPerThread / 32; ++c)
                tmem_ld_32x32(tmem_base + ((quarter * 32u) << 16) + buf * kBN + half * kColsPerThread + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&acc[c * 32]));
#pragma unroll
            for (int c = 0; c < kColsPerThread / 32; ++c) tmem_ld_wait_for(*reinterpret_cast<uint32_t(*)[32]>(&acc[c * 32]));
            tc_fence_before_sync();
            mbar_arrive(tmem_empty_bar(buf));
            store_rows<kBf16, kColsPerThread>(acc, p, dest, nt * kBN + half * kColsPerThread, staging, P::kStagingPitch, lane);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem_base, kTmemCols);
    }
}

template <int kBN, int kStages, bool kBf16>
cudaError_t launch(const MxGemmDev &dev, uint64_t max_tiles, cudaStream_t stream) {
    using P = Plan<kBN, kStages>;
    auto kernel = gemm_mx_kernel<kBN, kStages, kBf16>;
    static bool configured[64] = {false};
    int d = 0;
    cudaGetDevice(&d);
    if (d >= 0 && d < 64 && !configured[d]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kTotal);
        if (e != cudaSuccess) return e;
        configured[d] = true;
    }
    int sms = 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, d);
    if (sms <= 0) sms = 148;
    if (sm_budget() > 0 && sm_budget() < sms) sms = sm_budget();
    const uint32_t grid = (uint32_t)(max_tiles < (uint64_t)sms ? max_tiles : (uint64_t)sms);
    kernel<<<grid, kThreads, P::kTotal, stream>>>(dev);
    return cudaGetLastError();
}

} // namespace

cudaError_t launch_gemm_mx(const MxGemmArgs &args, cudaStream_t stream) {
    if (args.m == 0 || args.n == 0) return cudaSuccess;
    if (args.m > 0x7fffff00ull || args.n > 0x7fffff00ull || args.k > 0x7fffff00ull) return cudaErrorInvalidValue;
    constexpr int kBN = 128, kStages = 5;
    MxGemmDev dev;
    dev.a_chunks = static_cast<const uint8_t *>(args.a_chunks);
    dev.b_chunks = static_cast<const uint8_t *>(args.b_chunks);
    dev.c = static_cast<uint8_t *>(args.c);
    dev.c_stride = args.c_stride;
    dev.m = (uint32_t)args.m;
    dev.n = (uint32_t)args.n;
    dev.kblocks = (uint32_t)((args.k + kMxChunkValues - 1) / kMxChunkValues);
    dev.group_blocks = (uint32_t)((args.n + kChunkRows - 1) / kChunkRows);
    dev.tiles_m = (uint32_t)((args.m + kBM - 1) / kBM);
    dev.tiles_n = (uint32_t)((args.n + kBN - 1) / kBN);
    dev.tiles = args.tiles;
    dev.tile_count = args.tile_count;
    dev.row_dest = args.row_dest;
    dev.error_word = args.error_word;
    wait_limits_us(dev.wait_us);
    const uint64_t tiles = (args.tiles ? args.max_tiles : dev.tiles_m) * (uint64_t)dev.tiles_n;
    if (tiles > 0x7fffffffull) return cudaErrorInvalidValue;
    return args.c_bf16 ? launch<kBN, kStages, true>(dev, tiles, stream) : launch<kBN, kStages, false>(dev, tiles, stream);
}

} // namespace nkb
