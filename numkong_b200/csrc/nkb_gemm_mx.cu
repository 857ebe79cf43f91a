// Product of two MXFP4 operands in tile form (nkb_mx.h): C = A . B^T with f32 accumulation, f32 or bf16 cells, one packed
// matrix or a group of them.
//
//   C[i, j] = sum over blocks b of 2^(sa[i,b] + sb[j,b] - 254) * sum over the block's 32 values of a_l b_l
//
// tcgen05.mma.kind::mxf4 takes 64 values of depth a step and applies the scales inside: the scales come from TMEM. Four warps,
// one for each 32-lane quarter, bring a chunk's scale tiles there through registers (tcgen05.st) beside the MMAs. tcgen05.cp would
// bring them from shared memory in one instruction, but runs in the queue of the MMAs and costs them about 46 cycles a tile.
// e2m1 products are multiples of 1/4 of at most 36, so the sum of a block of 32 is a multiple of 1/4 of at most 1152 and exact. Over the
// depth the f32 accumulator holds 2^24 of the smallest block's quarters: sums stay exact while 4608 times the blocks times the ratio of
// the largest to the smallest product of scales stays below that, at worst a ratio of 2^3 at a depth of 8192; beyond, each step adds the
// roundings of an f32 sum.
//
// One persistent CTA per SM: warp 0 brings B to shared memory with untiled bulk copies and warp 14 brings A, warp 1 issues the MMAs,
// warps 2..9 read the accumulators out and store the cells, warps 10..13 store scales.
#include <cuda_bf16.h>
#include <type_traits>
#include "nkb_mx.h"
#include "nkb_mx_encode.cuh"
#include "nkb_ptx.cuh"

namespace nkb {

namespace {

constexpr int kBM = 128;
constexpr int kEpilogueWarps = 8;
constexpr int kScaleWarps = 4;
constexpr int kThreads = 64 + 32 * (kEpilogueWarps + kScaleWarps + 1);
constexpr int kSecondLoader = 2 + kEpilogueWarps + kScaleWarps;  // warp that fetches A
constexpr uint32_t kGroupM = 8;      // row tiles walked before the next column tile

struct MxGemmDev {
    const uint8_t *a_codes, *a_scales;  // tile form: codes and scales of the first chunk; with a_row_major only the scales
    const uint8_t *b_codes, *b_scales;
    uint8_t *c;
    uint64_t c_stride;
    uint32_t m, n, kblocks;
    uint32_t tiles_m, tiles_n;
    uint32_t group_blocks;           // row blocks of 128 per packed matrix
    const MxRowTile *tiles;
    const int32_t *tile_count, *row_dest;
    uint32_t tiles_fresh;            // the tiles are written by the kernel before, like A
    uint32_t a_row_major;            // A's codes are read from the caller's rows
    uint32_t a_blocks;               // row blocks A's buffers hold
    const uint8_t *x;                // float rows of A the kernel quantises itself, their stride, type and length
    uint64_t x_stride;
    uint32_t x_type, k;
    unsigned int *error_word;
    uint32_t wait_us[kWaitSites];
};

// Shared memory of the single-CTA kernel: a ring of stages with the codes of A and B, and a ring of groups of four chunks' scales
// (a bulk copy costs its issuer about 110 cycles whatever its size, so scales come four chunks at a time). The MMA always reads 128 rows of
// A; with kARows = 16 a stage holds 16 of them and the rest of what it reads is the stages behind (and 14 KiB of slack): rows of the
// accumulator nobody looks at. That leaves room for more stages of B, which is what a product with few rows waits for.
constexpr uint32_t kScaleGroup = 4, kScaleRing = 3;
template <int kBN, int kARows>
struct Plan {
    static constexpr int kABytes = kARows * 128, kBBytes = kBN * 128;
    static constexpr int kScaleBytes = kScaleRing * 2 * kScaleGroup * kMxScaleBytes;  // per group: A's tiles, B's tiles
    static constexpr int kStagingPitch = 144;  // bytes per staged row: 128 and one 16-byte piece against bank conflicts
    static constexpr int kStagingBytes = kEpilogueWarps * 32 * kStagingPitch;
    static constexpr int kRoom = 227 * 1024 - 1024 - 512 - kStagingBytes - kScaleBytes - (kBM - kARows) * 128;
    static constexpr int kStages = kRoom / (kBBytes + kABytes) < 16 ? kRoom / (kBBytes + kABytes) : 16;
    static constexpr int kBRing = kStages * kABytes + (kBM - kARows) * 128;
    static constexpr int kScaleOffset = kBRing + kStages * kBBytes;
    static constexpr int kBarrierOffset = kScaleOffset + kScaleBytes;
    static constexpr int kStagingOffset = kBarrierOffset + 512;
    static constexpr int kTotal = kStagingOffset + kStagingBytes + 1024;
    static_assert(kBRing % 1024 == 0 && kTotal <= 227 * 1024, "aligned operands that fit");
};

__device__ __forceinline__ void tile_coords(uint32_t tile, uint32_t tiles_m, uint32_t tiles_n, uint32_t &mt, uint32_t &nt) {
    const uint32_t per_group = kGroupM * tiles_n, group = tile / per_group, first = group * kGroupM;
    const uint32_t rows = min(tiles_m - first, kGroupM), in_group = tile % per_group;
    mt = first + in_group % rows;
    nt = in_group / rows;
    if (group & 1u) nt = tiles_n - 1u - nt;  // the packed rows touched last are still in L2
}

// Stores this thread's row x kCols f32 accumulators: up to 128 bytes of a row at a time go through the warp's staging block, so that
// a store instruction writes whole lines. `dest` is this lane's destination row, negative for none. Rows that do not lie on 16-byte
// boundaries (an odd width): f32 goes out a row at a time, one cell per lane; a bf16 row is staged as far off its boundary as it is in
// memory, so that seven of its pieces still go out as 16 bytes, the two at its ends in words and, where it begins in the middle of a
// word, two single cells. 1000 x 5003 x 2500 bf16: 27 us with words throughout, 20 us so; f32: 25 us so, 21 us a row at a time.
template <bool kBf16, int kCols>
__device__ __forceinline__ void store_rows(const uint32_t (&acc)[kCols], const MxGemmDev &p, int64_t dest, uint32_t col_base, uint8_t *staging, int pitch, int lane) {
    constexpr int kCell = kBf16 ? 2 : 4;
    constexpr int kPieceCols = kCols * kCell < 128 ? kCols : 128 / kCell;
    constexpr int kWords = kPieceCols * kCell / 4, kQuads = kWords / 4;  // words and 16-byte parts of a staged row
    static_assert(kCols % kPieceCols == 0 && kQuads >= 2, "whole pieces");
    if (!__any_sync(0xffffffffu, dest >= 0)) return;
    uint8_t *const my_row = dest >= 0 ? p.c + (uint64_t)dest * p.c_stride : nullptr;
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.c) | p.c_stride) & 15u) == 0;
    auto of_lane = [](uint8_t *ptr, int from) {
        return reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(ptr), from));
    };
#pragma unroll
    for (int c = 0; c < kCols / kPieceCols; ++c) {
        const uint32_t col0 = col_base + c * kPieceCols;
        if (col0 >= p.n) break;
        uint32_t words[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (kBf16) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(__uint_as_float(acc[c * kPieceCols + 2 * i]), __uint_as_float(acc[c * kPieceCols + 2 * i + 1]));
                words[i] = *reinterpret_cast<const uint32_t *>(&two);
            } else {
                words[i] = acc[c * kPieceCols + i];
            }
        }
        const uint32_t cells = min((uint32_t)kPieceCols, p.n - col0);
        uint8_t *const mine = my_row ? my_row + (uint64_t)col0 * kCell : nullptr;
        if (!kBf16 || aligned || cells != kPieceCols) {
#pragma unroll
            for (int q = 0; q < kQuads; ++q)
                *reinterpret_cast<uint4 *>(staging + lane * pitch + q * 16) = make_uint4(words[4 * q], words[4 * q + 1], words[4 * q + 2], words[4 * q + 3]);
            __syncwarp();
            if (!kBf16 && !aligned) {
#pragma unroll 8
                for (int r = 0; r < 32; ++r) {
                    uint8_t *row = of_lane(mine, r);
                    if (row && (uint32_t)lane < cells) reinterpret_cast<uint32_t *>(row)[lane] = reinterpret_cast<const uint32_t *>(staging + r * pitch)[lane];
                }
            } else if (cells == kPieceCols) {
#pragma unroll
                for (int it = 0; it < kQuads; ++it) {
                    const int r = it * (32 / kQuads) + lane / kQuads, q = lane % kQuads;
                    uint8_t *row = of_lane(mine, r);
                    if (row) __stcs(reinterpret_cast<uint4 *>(row) + q, *reinterpret_cast<const uint4 *>(staging + r * pitch + q * 16));
                }
            } else {  // the last columns
                for (int r = 0; r < 32; ++r) {
                    uint8_t *row = of_lane(mine, r);
                    for (uint32_t i = lane; row && i < cells; i += 32) {
                        if constexpr (kBf16) reinterpret_cast<uint16_t *>(row)[i] = reinterpret_cast<const uint16_t *>(staging + r * pitch)[i];
                        else reinterpret_cast<uint32_t *>(row)[i] = reinterpret_cast<const uint32_t *>(staging + r * pitch)[i];
                    }
                }
            }
        } else {
            const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(mine) & 15u;
            const bool odd = off & 2u;  // the row begins in the middle of a word
            uint32_t *to = reinterpret_cast<uint32_t *>(staging + lane * pitch) + off / 4;
#pragma unroll
            for (int i = 0; i <= kWords; ++i) {
                const uint32_t low = i > 0 ? words[i > 0 ? i - 1 : 0] : 0u, high = i < kWords ? words[i < kWords ? i : 0] : 0u;
                to[i] = odd ? __funnelshift_l(low, high, 16) : high;
            }
            __syncwarp();
#pragma unroll
            for (int it = 0; it < kQuads; ++it) {
                const int r = it * (32 / kQuads) + lane / kQuads, q = lane % kQuads;
                uint8_t *row = of_lane(mine, r);
                const uintptr_t at = reinterpret_cast<uintptr_t>(row);
                if (row && (q > 0 || (at & 15u) == 0))
                    __stcs(reinterpret_cast<uint4 *>(at & ~(uintptr_t)15) + q, *reinterpret_cast<const uint4 *>(staging + r * pitch + q * 16));
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {  // four lanes a row: a word each, of the first piece or of the one behind the last
                const int r = it * 8 + lane / 4;
                const uint32_t j = lane % 4;
                uint8_t *row = of_lane(mine, r);
                const uint32_t o = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
                uint32_t *base = reinterpret_cast<uint32_t *>(reinterpret_cast<uintptr_t>(row) & ~(uintptr_t)15);
                const uint32_t *from = reinterpret_cast<const uint32_t *>(staging + r * pitch);
                if (row && o != 0) {
                    if (j >= (o + 3) / 4) base[j] = from[j];
                    else if (j < o / 4) base[kWords + j] = from[kWords + j];
                    else {  // shared with the cell before the row's first, and with the one behind its last
                        reinterpret_cast<uint16_t *>(base + j)[1] = (uint16_t)(from[j] >> 16);
                        reinterpret_cast<uint16_t *>(base + kWords + j)[0] = (uint16_t)from[kWords + j];
                    }
                }
            }
        }
        __syncwarp();
    }
}

// The (tile, depth block) sequence of one CTA or CTA pair out of `step`, with the rows and the packed matrix of its tile.
template <int kTileRows>
struct Walk {
    const MxGemmDev &p;
    uint32_t tile, kb, mt, nt, tiles_m, step, rows, group;
    __device__ Walk(const MxGemmDev &p_, uint32_t first, uint32_t step_, uint32_t tiles_m_)
        : p(p_), tile(first), kb(0), mt(0), nt(0), tiles_m(tiles_m_), step(step_), rows(0), group(0) { locate(); }
    __device__ bool valid() const { return tile < tiles_m * p.tiles_n; }
    __device__ void locate() {
        if (!valid()) return;
        tile_coords(tile, tiles_m, p.tiles_n, mt, nt);
        if (p.tiles) {
            const int2 t = *reinterpret_cast<const int2 *>(p.tiles + mt);
            group = (uint32_t)t.x;
            rows = (uint32_t)t.y;
        } else {
            rows = min(p.m - mt * kTileRows, (uint32_t)kTileRows);
        }
    }
    __device__ void next_tile() {
        kb = 0;
        tile += step;
        locate();
    }
    __device__ void next() {
        if (++kb == p.kblocks) next_tile();
    }
};

// Eight values of row `row` from `first` on, zeros past the end.
template <uint32_t kType>
__device__ __forceinline__ void load_row8(const MxGemmDev &p, uint32_t row, uint32_t first, uint4 (&raw)[2]) {
    constexpr int kBytes = kType == kF32 ? 4 : 2;
    const uint8_t *from = p.x + row * p.x_stride + (uint64_t)first * kBytes;
    raw[0] = raw[1] = make_uint4(0, 0, 0, 0);
    if (first + 8 <= p.k && (reinterpret_cast<uintptr_t>(from) & 15u) == 0) {
        raw[0] = __ldg(reinterpret_cast<const uint4 *>(from));
        if constexpr (kType == kF32) raw[1] = __ldg(reinterpret_cast<const uint4 *>(from) + 1);
    } else {
        uint32_t w[8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + i < p.k) {
                if constexpr (kType == kF32) w[i] = __ldg(reinterpret_cast<const uint32_t *>(from) + i);
                else w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(from) + i) << (16 * (i & 1));
            }
        raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
        raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}
template <uint32_t kType>
__device__ __forceinline__ uint32_t quantise_row8(const uint4 (&raw)[2], uint32_t &scale) {
    float v[8];
    uint32_t largest;
    if constexpr (kType == kF32) largest = unpack8<kType>(raw, v);
    else largest = unpack8<kType>({raw[0]}, v);
    return quantise8(v, largest, scale);
}

// With kOwnA the epilogue warps quantise A's one or two rows into the rings while the packed matrix streams in, every eighth chunk each:
// one launch and no workspace, at the price of every CTA doing it again.
constexpr uint32_t kOwnRows = 2;
template <int kBN, int kARows, bool kOwnA, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1) gemm_mx_kernel(const MxGemmDev p) {
    using P = Plan<kBN, kARows>;
    constexpr int kStages = P::kStages;
    constexpr int kColsPerThread = kBN / 2;
    constexpr int kScaleCols = 16;  // one chunk's scales: eight columns for 128 rows of A, eight for the row block of B
    static_assert(2 * kBN + kStages * kScaleCols <= 512, "two accumulators and every stage's scales fit TMEM");
    static_assert(kBN == 64 || kBN == 128, "a tile's scales begin on an even TMEM column");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bar_base = smem_base + P::kBarrierOffset;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
    auto scale_full_bar = [&](uint32_t g) { return bar_base + 8u * (2 * kStages + g); };
    auto scale_empty_bar = [&](uint32_t g) { return bar_base + 8u * (2 * kStages + kScaleRing + g); };
    auto tmem_full_bar = [&](int a) { return bar_base + 8u * (2 * kStages + 2 * kScaleRing + a); };
    auto tmem_empty_bar = [&](int a) { return bar_base + 8u * (2 * kStages + 2 * kScaleRing + 2 + a); };
    const uint32_t drain_bar = bar_base + 8u * (2 * kStages + 2 * kScaleRing + 4);
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + P::kBarrierOffset + 8 * (2 * kStages + 2 * kScaleRing + 5));
    static_assert(8 * (2 * kStages + 2 * kScaleRing + 6) <= 512, "barriers fit");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        // A stage is full when B's loader, A's loader or quantiser and the scale warps have arrived.
        constexpr uint32_t fillers = 2 + kScaleWarps;
        for (int s = 0; s < kStages; ++s) { mbar_init(full_bar(s), fillers); mbar_init(empty_bar(s), 1); }
        for (uint32_t g = 0; g < kScaleRing; ++g) { mbar_init(scale_full_bar(g), kOwnA ? 1 + kEpilogueWarps : 2); mbar_init(scale_empty_bar(g), kScaleWarps); }
        for (int a = 0; a < 2; ++a) { mbar_init(tmem_full_bar(a), 1); mbar_init(tmem_empty_bar(a), kEpilogueWarps * 32); }
        mbar_init(drain_bar, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t *>(tmem_slot)), 512);
        tmem_relinquish<1>();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    if (p.tiles_fresh) wait_for_previous_kernel();
    const uint32_t tiles_m = p.tile_count ? (uint32_t)*p.tile_count : p.tiles_m;

    // One loader for each operand: its scales four chunks at a time, its codes chunk by chunk.
    auto run_loader = [&](uint32_t scale_part, auto scale_source, auto code_bytes, auto code_copy) {
        int stage = 0;
        uint32_t phase = 0, group = 0, group_phase = 0, issued = 0, groups = 0;
        bool ok = true;
        for (Walk<kBM> w(p, blockIdx.x, gridDim.x, tiles_m); w.valid(); w.next()) {
            if (w.kb % kScaleGroup == 0) {
                if (!mbar_wait(scale_empty_bar(group), group_phase ^ 1u, 1, p.error_word, p.wait_us[1])) { ok = false; break; }
                const uint32_t bytes = min(kScaleGroup, p.kblocks - w.kb) * kMxScaleBytes;
                mbar_expect_tx(scale_full_bar(group), bytes);
                bulk_load(smem_base + P::kScaleOffset + (2 * group + scale_part) * kScaleGroup * kMxScaleBytes, scale_source(w), bytes, scale_full_bar(group));
                ++groups;
                if (++group == kScaleRing) { group = 0; group_phase ^= 1u; }
            }
            if (!mbar_wait(empty_bar(stage), phase ^ 1u, 1, p.error_word, p.wait_us[1])) { ok = false; break; }
            mbar_expect_tx(full_bar(stage), code_bytes(w));
            code_copy(w, stage);
            ++issued;
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) {  // copies in flight must land before the block may retire
            for (uint32_t i = 0; i < issued && i < (uint32_t)kStages; ++i) {
                if (stage == 0) { stage = kStages; phase ^= 1u; }
                --stage;
                if (!mbar_wait(full_bar(stage), phase, 6, p.error_word, p.wait_us[6])) break;
            }
            for (uint32_t i = 0; i < groups && i < kScaleRing; ++i) {
                if (group == 0) { group = kScaleRing; group_phase ^= 1u; }
                --group;
                if (!mbar_wait(scale_full_bar(group), group_phase, 6, p.error_word, p.wait_us[6])) break;
            }
        }
    };

    if (warp == 0) {
        // The packed matrix does not depend on the kernel before, which may still be quantising A.
        if (lane == 0) {
            auto chunk = [&](const Walk<kBM> &w) { return ((uint64_t)w.group * p.group_blocks + w.nt * kBN / 128u) * p.kblocks + w.kb; };
            run_loader(1, [&](const Walk<kBM> &w) { return p.b_scales + chunk(w) * kMxScaleBytes; }, [&](const Walk<kBM> &) { return (uint32_t)P::kBBytes; },
                       [&](const Walk<kBM> &w, int stage) {
                           bulk_load(smem_base + P::kBRing + stage * P::kBBytes, p.b_codes + chunk(w) * kMxCodeBytes + w.nt * kBN % 128u * 128u, P::kBBytes, full_bar(stage));
                       });
        }
    } else if (warp == kSecondLoader) {
        if (!kOwnA && lane == 0) {
            wait_for_previous_kernel();
            auto chunk = [&](const Walk<kBM> &w) { return (uint64_t)w.mt * p.kblocks + w.kb; };
            auto bytes = [&](const Walk<kBM> &w) { return (w.rows + 7u) / 8u * 1024u; };  // the row groups of eight that hold valid rows
            run_loader(0, [&](const Walk<kBM> &w) { return p.a_scales + chunk(w) * kMxScaleBytes; }, bytes,
                       [&](const Walk<kBM> &w, int stage) { bulk_load(smem_base + stage * P::kABytes, p.a_codes + chunk(w) * kMxCodeBytes, bytes(w), full_bar(stage)); });
        }
    } else if (warp == 1) {
        // The whole warp walks, one lane issues (see elect_one).
        uint32_t stage = 0, phase = 0, seq = 0;
        bool ok = true;
        const uint32_t num_tiles = tiles_m * p.tiles_n;
        for (uint32_t tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++seq) {
            uint32_t mt, nt;
            tile_coords(tile, tiles_m, p.tiles_n, mt, nt);
            const uint32_t b_column = 8u + nt * kBN % 128u / 32u;  // the tile's rows inside the row block's scales
            const uint32_t buf = seq & 1u, buf_phase = (seq >> 1) & 1u;
            if (!__all_sync(0xffffffffu, mbar_wait(tmem_empty_bar(buf), buf_phase ^ 1u, 2, p.error_word, p.wait_us[2]))) { ok = false; break; }
            tc_fence_after_sync();
            const uint32_t d_tmem = tmem_base + buf * kBN;
            for (uint32_t kb = 0; kb < p.kblocks; ++kb) {
                if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, 3, p.error_word, p.wait_us[3]))) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t scales = tmem_base + 2 * kBN + stage * kScaleCols;
                const uint64_t a_desc = make_smem_desc_sw128(smem_base + stage * P::kABytes), b_desc = make_smem_desc_sw128(smem_base + P::kBRing + stage * P::kBBytes);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_mxf4<1>(d_tmem, a_desc + 2u * k, b_desc + 2u * k, make_idesc_mxf4(kBM, kBN, (k & 1) * 2), scales + (k >> 1) * 4,
                                     scales + b_column + (k >> 1) * 4, (kb | (uint32_t)k) != 0u);
                    umma_commit(empty_bar(stage));
                    if (kb + 1 == p.kblocks) umma_commit(tmem_full_bar(buf));
                }
                __syncwarp();
                if (++stage == kStages) { stage = 0; phase ^= 1u; }
            }
        }
        if (elect_one()) umma_commit(drain_bar);  // shared memory and TMEM are released below: the last MMAs must have retired
        __syncwarp();
        mbar_wait(drain_bar, 0u, 5, p.error_word, p.wait_us[5]);
        __syncwarp();
    } else if (warp >= 2 + kEpilogueWarps) {
        // ------------------------------------------------------------ scales: shared memory -> this warp's 32-lane quarter of TMEM
        // A stage has TMEM columns of its own, free again when the stage is.
        const uint32_t column = tmem_base + (((uint32_t)warp & 3u) * 32u << 16) + 2 * kBN;
        int stage = 0;
        uint32_t phase = 0, group = 0, group_phase = 0;
        for (Walk<kBM> w(p, blockIdx.x, gridDim.x, tiles_m); w.valid(); w.next()) {
            const uint32_t in_group = w.kb % kScaleGroup;
            bool ok = in_group != 0 || mbar_wait(scale_full_bar(group), group_phase, 3, p.error_word, p.wait_us[3]);
            ok = ok && mbar_wait(empty_bar(stage), phase ^ 1u, 2, p.error_word, p.wait_us[2]);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after_sync();
            const uint4 *tiles = reinterpret_cast<const uint4 *>(smem_gen + P::kScaleOffset + (2 * group * kScaleGroup + in_group) * kMxScaleBytes) + lane;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 lo = tiles[i * kScaleGroup * kMxScaleBytes / 16], hi = tiles[i * kScaleGroup * kMxScaleBytes / 16 + 32];
                const uint32_t words[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                tmem_st_32x8(column + stage * kScaleCols + i * 8, words);
            }
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            const bool last = in_group == kScaleGroup - 1 || w.kb + 1 == p.kblocks;
            if (lane == 0) {
                mbar_arrive(full_bar(stage));  // the stage's scales are in TMEM
                if (last) mbar_arrive(scale_empty_bar(group));
            }
            if (last && ++group == kScaleRing) { group = 0; group_phase ^= 1u; }
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
    } else {
        const uint32_t quarter = warp & 3u, half = (uint32_t)(warp - 2) >> 2;
        uint8_t *staging = smem_gen + P::kStagingOffset + (warp - 2) * 32 * P::kStagingPitch;
        uint32_t seq = 0, phase = 0, group = 0, group_phase = 0, chunk = 0;
        int stage = 0;
        for (Walk<kBM> w(p, blockIdx.x, gridDim.x, tiles_m); w.valid(); w.next_tile(), ++seq) {
            if constexpr (kOwnA) {
                constexpr uint32_t kSets = kEpilogueWarps;
                const uint32_t set = (uint32_t)warp - 2u;
                auto own = [&](auto type) {
                    constexpr uint32_t kType = decltype(type)::value;
                    uint4 raw[kOwnRows][2];
                    auto fetch = [&](uint32_t kb) {
#pragma unroll
                        for (uint32_t r = 0; r < kOwnRows; ++r)
                            if (r < p.m && kb < p.kblocks) load_row8<kType>(p, r, kb * kMxChunkValues + lane * 8, raw[r]);
                    };
                    fetch((set + kSets - chunk % kSets) % kSets);  // the first chunk of the tile that is this warp's
                    for (uint32_t kb = 0; kb < p.kblocks; ++kb, ++chunk) {
                        const uint32_t in_group = kb % kScaleGroup;
                        bool ok = in_group != 0 || mbar_wait(scale_empty_bar(group), group_phase ^ 1u, 1, p.error_word, p.wait_us[1]);
                        const bool mine = chunk % kSets == set;
                        if (ok && mine) ok = mbar_wait(empty_bar(stage), phase ^ 1u, 1, p.error_word, p.wait_us[1]);
                        if (!__all_sync(0xffffffffu, ok)) return false;
                        if (mine) {
                            uint8_t *codes = smem_gen + stage * P::kABytes, *scales = smem_gen + P::kScaleOffset + (2 * group * kScaleGroup + in_group) * kMxScaleBytes;
#pragma unroll
                            for (uint32_t r = 0; r < kOwnRows; ++r) {
                                if (r >= p.m) continue;
                                uint32_t s;
                                const uint32_t word = quantise_row8<kType>(raw[r], s);
                                *reinterpret_cast<uint32_t *>(codes + r * 128u + ((((uint32_t)lane >> 2) ^ (r & 7u)) << 4) + (lane & 3) * 4) = word;
                                if ((lane & 3) == 0) scales[(lane >> 4) * 512 + r * 16 + ((lane >> 2) & 3)] = (uint8_t)s;
                            }
                            fetch(kb + kSets);
                            fence_proxy_async_smem();  // the MMA reads the codes through the other proxy
                            __syncwarp();
                            if (lane == 0) mbar_arrive(full_bar(stage));
                        }
                        if (in_group == kScaleGroup - 1 || kb + 1 == p.kblocks) {
                            __syncwarp();
                            if (lane == 0) mbar_arrive(scale_full_bar(group));
                            if (++group == kScaleRing) { group = 0; group_phase ^= 1u; }
                        }
                        if (++stage == kStages) { stage = 0; phase ^= 1u; }
                    }
                    return true;
                };
                const bool ok = p.x_type == kBF16 ? own(std::integral_constant<uint32_t, kBF16>{})
                                : p.x_type == kF16 ? own(std::integral_constant<uint32_t, kF16>{}) : own(std::integral_constant<uint32_t, kF32>{});
                if (!ok) break;
            }
            const uint32_t buf = seq & 1u, buf_phase = (seq >> 1) & 1u, in_tile = quarter * 32u + lane;
            int64_t dest = -1;
            if (in_tile < w.rows) dest = p.row_dest ? (int64_t)p.row_dest[(uint64_t)w.mt * kBM + in_tile] : (int64_t)w.mt * kBM + in_tile;
            // The whole warp leaves together: the stores below synchronise it.
            if (!__all_sync(0xffffffffu, mbar_wait(tmem_full_bar(buf), buf_phase, 4, p.error_word, p.wait_us[4]))) break;
            tc_fence_after_sync();
            uint32_t acc[kColsPerThread];
            const uint32_t from = tmem_base + ((quarter * 32u) << 16) + buf * kBN + half * kColsPerThread;
#pragma unroll
            for (int c = 0; c < kColsPerThread / 32; ++c) tmem_ld_32x32(from + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&acc[c * 32]));
#pragma unroll
            for (int c = 0; c < kColsPerThread / 32; ++c) tmem_ld_wait_for(*reinterpret_cast<uint32_t(*)[32]>(&acc[c * 32]));
            tc_fence_before_sync();
            mbar_arrive(tmem_empty_bar(buf));
            store_rows<kBf16, kColsPerThread>(acc, p, dest, w.nt * kBN + half * kColsPerThread, staging, P::kStagingPitch, lane);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------------------------------------
// CTA pairs (cta_group::2): two CTAs on neighbouring SMs share a 256 x 256 tile. Each loads its own 128 rows of A and half of
// B's rows; the leader issues. All loads count on the leader's barriers, hence tensor maps: chunks seen as rows of 128 bytes. Every
// CTA applies the scales of all of B's rows to its own half of the accumulator.
//
// TMEM holds two accumulators of 256 columns and the scales by letting the accumulators overlap: [0, 256) and
// [512 - scales - 256, 512 - scales). The epilogue reads the columns they share first and then lets the next tile's MMAs
// start, so they wait for a part of a read-out instead of all of it.
//
// Scales come by bulk copies, four chunks at a time, into a ring of their own. 8192 x 8192 x 8192 with the scale warps loading them from
// global memory instead: 277 us, since their loads wait behind the stores of the epilogue; with tcgen05.cp, six tiles a chunk: 253 us.
constexpr int kPairStages = 5;
constexpr int kPairScaleCols = 24;                                // 8 for 128 rows of A, 16 for 256 of B
constexpr int kPairSecond = 512 - 2 * kPairScaleCols - 256;       // first column of the second accumulator; two chunks' scales behind it
constexpr int kPairBOffset = kBM * 128;
constexpr int kPairStageBytes = 2 * kBM * 128;                    // A codes, B codes
constexpr uint32_t kPairScaleRing = 2;                            // groups of four chunks' scales: A's tiles, both row blocks of B
constexpr int kPairGroupBytes = 3 * kScaleGroup * kMxScaleBytes;
constexpr int kPairScaleOffset = kPairStages * kPairStageBytes;
constexpr int kPairBarrierOffset = kPairScaleOffset + kPairScaleRing * kPairGroupBytes;
constexpr int kPairStagingPitch = 144;
constexpr int kPairStagingOffset = kPairBarrierOffset + 256;
constexpr int kPairSmem = kPairStagingOffset + kEpilogueWarps * 32 * kPairStagingPitch + 1024;
static_assert(kPairSmem <= 227 * 1024, "one CTA per SM");
static_assert(kPairSecond >= 256 - 64, "the shared columns are the last / first 64 of the two accumulators at most");

struct PairMaps {
    CUtensorMap a, b;
};

template <bool kBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gemm_mx_pair_kernel(const __grid_constant__ PairMaps maps, const MxGemmDev p) {
    constexpr int kStages = kPairStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bar_base = smem_base + kPairBarrierOffset;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
    auto tmem_full_bar = [&](int a) { return bar_base + 8u * (2 * kStages + a); };
    const uint32_t shared_read_bar = bar_base + 8u * (2 * kStages + 4);  // the tile before is read, of this one the shared columns
    const uint32_t drain_bar = bar_base + 8u * (2 * kStages + 5);
    auto scale_full_bar = [&](uint32_t g) { return bar_base + 8u * (2 * kStages + 6 + g); };
    auto scale_empty_bar = [&](uint32_t g) { return bar_base + 8u * (2 * kStages + 6 + kPairScaleRing + g); };
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + kPairBarrierOffset + 8 * (2 * kStages + 6 + 2 * kPairScaleRing));
    static_assert(8 * (2 * kStages + 7 + 2 * kPairScaleRing) <= 256, "barriers fit");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    if (p.tiles_fresh) wait_for_previous_kernel();
    const uint32_t tiles_m = p.tile_count ? (uint32_t)*p.tile_count : p.tiles_m, num_tiles = tiles_m * p.tiles_n;
    if (threadIdx.x == 0) {
        prefetch_tensormap(&maps.a);
        prefetch_tensormap(&maps.b);
        for (int s = 0; s < kStages; ++s) { mbar_init(full_bar(s), 1 + 2 * kScaleWarps); mbar_init(empty_bar(s), 1); }  // copies and both CTAs' scales
        for (int a = 0; a < 2; ++a) mbar_init(tmem_full_bar(a), 1);
        for (uint32_t g = 0; g < kPairScaleRing; ++g) { mbar_init(scale_full_bar(g), 1); mbar_init(scale_empty_bar(g), kScaleWarps); }
        mbar_init(shared_read_bar, 2 * kEpilogueWarps);
        mbar_init(drain_bar, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(const_cast<uint32_t *>(tmem_slot)), 512);
        tmem_relinquish<2>();
    }
    tc_fence_before_sync();
    __syncwarp();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0, issued = 0;
            bool ok = true;
            wait_for_previous_kernel();
            for (Walk<256> w(p, pair, num_pairs, tiles_m); w.valid(); w.next()) {
                if (!mbar_wait<true>(empty_bar(stage), phase ^ 1u, 1, p.error_word, p.wait_us[1])) { ok = false; break; }
                const uint32_t dst = smem_base + stage * kPairStageBytes, full = map_to_cta(full_bar(stage), 0);
                const bool second = w.rows > kBM;  // the follower's rows of A exist
                if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * kBM * 128 + (second ? 2 : 1) * kBM * 128);
                const uint32_t a_block = w.mt * 2u + rank, b_block = w.group * p.group_blocks + w.nt * 2u + rank;
                if (rank == 0 || second) {
                    if (p.a_row_major) tma_load_2d_pair(dst, &maps.a, (int)(w.kb * 128u), (int)(a_block * kBM), full);
                    else tma_load_2d_pair(dst, &maps.a, 0, (int)((a_block * p.kblocks + w.kb) * kBM), full);
                }
                tma_load_2d_pair(dst + kPairBOffset, &maps.b, 0, (int)((b_block * p.kblocks + w.kb) * kBM), full);
                ++issued;
                if (++stage == kStages) { stage = 0; phase ^= 1u; }
            }
            if (!ok) {
                // Both CTAs' copies count on the leader's barriers: the leader waits for them, the follower sleeps (its last
                // copy is at least one wait limit old, and neither CTA retires before the cluster barrier).
                if (rank == 0) {
                    int s = stage;
                    uint32_t ph = phase;
                    for (uint32_t i = 0; i < issued && i < (uint32_t)kStages; ++i) {
                        if (s == 0) { s = kStages; ph ^= 1u; }
                        --s;
                        if (!mbar_wait<true>(full_bar(s), ph, 6, p.error_word, p.wait_us[6])) break;
                    }
                } else {
                    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {  // the whole warp walks, one lane issues (see elect_one)
            uint32_t stage = 0, phase = 0, seq = 0, chunk = 0;
            bool ok = true;
            for (uint32_t tile = pair; tile < num_tiles && ok; tile += num_pairs, ++seq) {
                if (seq > 0 && !__all_sync(0xffffffffu, mbar_wait<true>(shared_read_bar, (seq - 1u) & 1u, 2, p.error_word, p.wait_us[2]))) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t buf = seq & 1u, d_tmem = tmem_base + buf * kPairSecond;
                for (uint32_t kb = 0; kb < p.kblocks; ++kb, ++chunk) {
                    if (!__all_sync(0xffffffffu, mbar_wait<true>(full_bar(stage), phase, 3, p.error_word, p.wait_us[3]))) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint32_t src = smem_base + stage * kPairStageBytes;
                    const uint64_t a_desc = make_smem_desc_sw128(src), b_desc = make_smem_desc_sw128(src + kPairBOffset);
                    const uint32_t scales_a = tmem_base + kPairSecond + 256 + (chunk & 1u) * kPairScaleCols, scales_b = scales_a + 8;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_mxf4<2>(d_tmem, a_desc + 2u * k, b_desc + 2u * k, make_idesc_mxf4(256, 256, (k & 1) * 2), scales_a + (k >> 1) * 4,
                                         scales_b + (k >> 1) * 8, (kb | (uint32_t)k) != 0u);
                        umma_commit_pair(empty_bar(stage), 3);
                        if (kb + 1 == p.kblocks) umma_commit_pair(tmem_full_bar(buf), 3);
                    }
                    __syncwarp();
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
            if (elect_one()) umma_commit_pair(drain_bar, 1);
            __syncwarp();
            mbar_wait<true>(drain_bar, 0u, 5, p.error_word, p.wait_us[5]);
            __syncwarp();
        }
    } else if (warp == kSecondLoader) {
        // ------------------------------------------------------------ scales of this CTA's rows of A and of all rows of B
        if (lane == 0) {
            wait_for_previous_kernel();
            const uint32_t a_last = p.a_blocks - 1, b_last = p.group_blocks - 1;
            uint32_t group = 0, phase = 0, groups = 0;
            bool ok = true;
            for (Walk<256> w(p, pair, num_pairs, tiles_m); w.valid() && ok; w.next_tile()) {
                const uint8_t *a = p.a_scales + (uint64_t)min(w.mt * 2u + rank, a_last) * p.kblocks * kMxScaleBytes;
                const uint8_t *b[2];
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) b[j] = p.b_scales + (uint64_t)(w.group * p.group_blocks + min(w.nt * 2u + j, b_last)) * p.kblocks * kMxScaleBytes;
                for (uint32_t kb = 0; kb < p.kblocks; kb += kScaleGroup) {
                    if (!mbar_wait(scale_empty_bar(group), phase ^ 1u, 1, p.error_word, p.wait_us[1])) { ok = false; break; }
                    const uint32_t bytes = min(kScaleGroup, p.kblocks - kb) * kMxScaleBytes, dst = smem_base + kPairScaleOffset + group * kPairGroupBytes;
                    mbar_expect_tx(scale_full_bar(group), 3 * bytes);
                    bulk_load(dst, a + (uint64_t)kb * kMxScaleBytes, bytes, scale_full_bar(group));
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j)
                        bulk_load(dst + (1 + j) * kScaleGroup * kMxScaleBytes, b[j] + (uint64_t)kb * kMxScaleBytes, bytes, scale_full_bar(group));
                    ++groups;
                    if (++group == kPairScaleRing) { group = 0; phase ^= 1u; }
                }
            }
            for (uint32_t i = 0; !ok && i < groups && i < kPairScaleRing; ++i) {  // copies in flight must land before the block may retire
                if (group == 0) { group = kPairScaleRing; phase ^= 1u; }
                --group;
                if (!mbar_wait(scale_full_bar(group), phase, 6, p.error_word, p.wait_us[6])) break;
            }
        }
    } else if (warp >= 2 + kEpilogueWarps) {
        // ------------------------------------------------------------ scales: shared memory -> this warp's 32-lane quarter of TMEM
        const uint32_t column = tmem_base + (((uint32_t)warp & 3u) * 32u << 16) + kPairSecond + 256;
        uint32_t chunk = 0, group = 0, group_phase = 0, freed_phase = 0;
        int stage = 0, freed = 0;  // of the chunk being stored, and of the one whose scales it overwrites
        for (Walk<256> w(p, pair, num_pairs, tiles_m); w.valid(); w.next(), ++chunk) {
            const uint32_t in_group = w.kb % kScaleGroup;
            if (in_group == 0 && !__all_sync(0xffffffffu, mbar_wait(scale_full_bar(group), group_phase, 3, p.error_word, p.wait_us[3]))) break;
            // Lane r of every quarter holds line r of each tile: A for both halves of the chunk's depth, B for both halves of its rows.
            const uint4 *tiles = reinterpret_cast<const uint4 *>(smem_gen + kPairScaleOffset + group * kPairGroupBytes + in_group * kMxScaleBytes) + lane;
            constexpr int kPart = kScaleGroup * kMxScaleBytes / 16;
            const uint4 r[6] = {tiles[0], tiles[32], tiles[kPart], tiles[2 * kPart], tiles[kPart + 32], tiles[2 * kPart + 32]};
            if (chunk >= 2) {  // the MMAs of two chunks ago have read theirs
                if (!__all_sync(0xffffffffu, mbar_wait<true>(empty_bar(freed), freed_phase, 2, p.error_word, p.wait_us[2]))) break;
                if (++freed == kStages) { freed = 0; freed_phase ^= 1u; }
                tc_fence_after_sync();
            }
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const uint32_t words[8] = {r[2 * i].x, r[2 * i].y, r[2 * i].z, r[2 * i].w, r[2 * i + 1].x, r[2 * i + 1].y, r[2 * i + 1].z, r[2 * i + 1].w};
                tmem_st_32x8(column + (chunk & 1u) * kPairScaleCols + i * 8, words);
            }
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            const bool last = in_group == kScaleGroup - 1 || w.kb + 1 == p.kblocks;
            if (lane == 0) {
                mbar_arrive_cluster_addr(map_to_cta(full_bar(stage), 0));
                if (last) mbar_arrive(scale_empty_bar(group));
            }
            if (last && ++group == kPairScaleRing) { group = 0; group_phase ^= 1u; }
            if (++stage == kStages) stage = 0;
        }
    } else {
        const uint32_t quarter = warp & 3u, half = (uint32_t)(warp - 2) >> 2;
        uint8_t *staging = smem_gen + kPairStagingOffset + (warp - 2) * 32 * kPairStagingPitch;
        uint32_t seq = 0;
        for (Walk<256> w(p, pair, num_pairs, tiles_m); w.valid(); w.next_tile(), ++seq) {
            const uint32_t buf = seq & 1u;
            const uint32_t in_tile = rank * 128u + quarter * 32u + lane;
            int64_t dest = -1;
            if (in_tile < w.rows) dest = p.row_dest ? (int64_t)p.row_dest[(uint64_t)w.mt * 256u + in_tile] : (int64_t)w.mt * 256u + in_tile;
            if (!__all_sync(0xffffffffu, mbar_wait<true>(tmem_full_bar(buf), (seq >> 1) & 1u, 4, p.error_word, p.wait_us[4]))) break;
            tc_fence_after_sync();
            // 64 columns at a time. Those shared with the other accumulator - the last of the first, the first of the second - come first.
            const uint32_t first = buf == 0 ? 64u : 0u;
            const bool shares = half == 1u - buf;
            auto arrive = [&]() {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_addr(map_to_cta(shared_read_bar, 0));
            };
            if (!shares) arrive();
#pragma unroll 1
            for (uint32_t part = 0; part < 2; ++part) {
                const uint32_t in_half = part == 0 ? first : 64u - first;
                uint32_t acc[64];
                const uint32_t from = tmem_base + ((quarter * 32u) << 16) + buf * kPairSecond + half * 128u + in_half;
                tmem_ld_32x32(from, *reinterpret_cast<uint32_t(*)[32]>(&acc[0]));
                tmem_ld_32x32(from + 32, *reinterpret_cast<uint32_t(*)[32]>(&acc[32]));
                tmem_ld_wait_for(*reinterpret_cast<uint32_t(*)[32]>(&acc[0]));
                tmem_ld_wait_for(*reinterpret_cast<uint32_t(*)[32]>(&acc[32]));
                if (shares && part == 0) arrive();
                store_rows<kBf16, 64>(acc, p, dest, w.nt * 256u + half * 128u + in_half, staging, kPairStagingPitch, lane);
            }
        }
    }
    tc_fence_before_sync();
    __syncwarp();
    cluster_sync_all();  // neither CTA retires while its partner reads its shared memory or signals its barriers
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<2>(tmem_base, 512);
    }
}

int sm_count() {
    static int cached[64] = {0};
    int d = 0;
    cudaGetDevice(&d);
    if (d < 0 || d >= 64) d = 0;
    if (!cached[d]) {
        int n = 0;
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d);
        cached[d] = n > 0 ? n : 148;
    }
    return cached[d];
}
int usable_sms() { return sm_budget() > 0 && sm_budget() < sm_count() ? sm_budget() : sm_count(); }

// Rows of 128 bytes, `box_rows` of them per copy.
bool line_map(CUtensorMap &map, const void *base, uint64_t lines, uint32_t box_rows) {
    cuuint64_t dims[2] = {128, lines};
    cuuint64_t strides[1] = {128};
    cuuint32_t box[2] = {128, box_rows}, steps[2] = {1, 1};
    return get_encode_tiled()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Launches as the dependent of the kernel before on the stream, which by construction is this library's own (it prepares A) and no
// dependent itself: everything before that one has finished.
template <typename... Args>
cudaError_t launch_dependent(void (*kernel)(Args...), uint32_t grid, int threads, int smem, cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <bool kBf16>
cudaError_t launch_pair(const PairMaps &maps, const MxGemmDev &dev, uint64_t tiles, cudaStream_t stream) {
    auto kernel = gemm_mx_pair_kernel<kBf16>;
    static int max_pairs[64] = {0};
    int d = 0;
    cudaGetDevice(&d);
    if (d < 0 || d >= 64) d = 0;
    if (max_pairs[d] == 0) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * (sm_count() / 2));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kPairSmem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) { cudaGetLastError(); n = sm_count() / 2; }
        max_pairs[d] = n;
    }
    uint32_t pairs = (uint32_t)(tiles < 0x7fffffffull ? tiles : 0x7fffffffull), most = (uint32_t)max_pairs[d];
    if (usable_sms() > 1 && (uint32_t)usable_sms() / 2 < most) most = (uint32_t)usable_sms() / 2;
    if (pairs > most) pairs = most;
    return launch_dependent(kernel, 2 * pairs, kThreads, kPairSmem, stream, maps, dev);
}

template <int kBN, int kARows, bool kOwnA, bool kBf16>
cudaError_t launch(const MxGemmDev &dev, uint64_t max_tiles, cudaStream_t stream) {
    using P = Plan<kBN, kARows>;
    auto kernel = gemm_mx_kernel<kBN, kARows, kOwnA, kBf16>;
    static bool configured[64] = {false};
    int d = 0;
    cudaGetDevice(&d);
    if (d >= 0 && d < 64 && !configured[d]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kTotal);
        if (e != cudaSuccess) return e;
        configured[d] = true;
    }
    const uint32_t grid = (uint32_t)(max_tiles < (uint64_t)usable_sms() ? max_tiles : (uint64_t)usable_sms());
    if constexpr (kOwnA) {
        kernel<<<grid, kThreads, P::kTotal, stream>>>(dev);
        return cudaGetLastError();
    } else {
        return launch_dependent(kernel, grid, kThreads, P::kTotal, stream, dev);
    }
}

template <int kARows, bool kOwnA>
cudaError_t launch_by_width(int bn, bool bf16, const MxGemmDev &dev, uint64_t max_tiles, cudaStream_t stream) {
    if (bn == 64) return bf16 ? launch<64, kARows, kOwnA, true>(dev, max_tiles, stream) : launch<64, kARows, kOwnA, false>(dev, max_tiles, stream);
    return bf16 ? launch<128, kARows, kOwnA, true>(dev, max_tiles, stream) : launch<128, kARows, kOwnA, false>(dev, max_tiles, stream);
}

} // namespace

// CTA pairs, when their tiles keep two thirds of the SMs busy. 2048^3 (64 tiles): 11.0 us against 13.5; 512 x 8192 x 8192 (64): 23.3 against
// 28.7; 1024 x 2048 x 4096 (32): 13.6 against 13.4; 256 x 8192 x 8192 (32): 20.4 against 16.9. Not for rows that one CTA's tile holds, for which
// the follower's half would be empty: 8 x 32768 x 4096 (128): 19.6 against 16.3; 128 x 32768 x 4096: 22.7 against 18.6.
bool gemm_mx_reads_rows(uint64_t m, uint64_t n, uint64_t) {
    return m > kBM && ((m + 255) / 256) * ((n + 255) / 256) >= (uint64_t)sm_count() / 3;
}

// Every CTA quantises the rows again, and with more than two a chunk took several warps, so that its loads no longer lay eight chunks ahead:
// 8 x 8192 x 8192 took 22.8 us inside and takes 13.2 us with a kernel before it; 1 x 4096 x 4096 takes 8.8 us inside, one launch.
bool gemm_mx_quantises(uint64_t m) { return m <= kOwnRows; }

cudaError_t launch_gemm_mx(const MxGemmArgs &args, cudaStream_t stream) {
    if (args.m == 0 || args.n == 0) return cudaSuccess;
    if (args.m > 0x7fffff00ull || args.n > 0x7fffff00ull || args.k > 0x7fffff00ull) return cudaErrorInvalidValue;
    if (args.x && (!gemm_mx_quantises(args.m) || args.tiles)) return cudaErrorInvalidValue;
    MxGemmDev dev;
    dev.kblocks = (uint32_t)((args.k + kMxChunkValues - 1) / kMxChunkValues);
    dev.group_blocks = (uint32_t)((args.n + kChunkRows - 1) / kChunkRows);
    const uint64_t a_blocks = args.tiles ? args.max_tiles * (args.tile_rows / kChunkRows) : (args.m + kBM - 1) / kBM;
    const uint64_t a_chunks = a_blocks * dev.kblocks, b_chunks = args.groups * dev.group_blocks * dev.kblocks;
    // Tensor maps address lines of 128 bytes with 31-bit coordinates; both kernels count chunks in 32 bits.
    if (a_blocks > 0x00ffffffull || a_chunks > 0x7fffff00ull / 128 || b_chunks > 0x7fffff00ull / 128) return cudaErrorInvalidValue;
    dev.a_codes = static_cast<const uint8_t *>(args.a_chunks);
    dev.a_scales = dev.a_codes + (args.a_codes ? 0 : a_chunks * kMxCodeBytes);
    dev.b_codes = static_cast<const uint8_t *>(args.b_chunks);
    dev.b_scales = dev.b_codes + b_chunks * kMxCodeBytes;
    dev.c = static_cast<uint8_t *>(args.c);
    dev.c_stride = args.c_stride;
    dev.m = (uint32_t)args.m;
    dev.n = (uint32_t)args.n;
    dev.tiles = args.tiles;
    dev.tile_count = args.tile_count;
    dev.tiles_fresh = args.tiles_fresh;
    dev.row_dest = args.row_dest;
    dev.x = static_cast<const uint8_t *>(args.x);
    dev.x_stride = args.x_stride;
    dev.x_type = args.x_type;
    dev.k = (uint32_t)args.k;
    dev.error_word = args.error_word;
    wait_limits_us(dev.wait_us);
    dev.a_row_major = args.a_codes != nullptr;
    dev.a_blocks = (uint32_t)a_blocks;
    if (args.tiles ? args.tile_rows == 256 : !args.x && gemm_mx_reads_rows(args.m, args.n, args.k)) {
        if (!get_encode_tiled()) return cudaErrorNotSupported;
        dev.tiles_m = (uint32_t)((args.m + 255) / 256);
        dev.tiles_n = (uint32_t)((args.n + 255) / 256);
        PairMaps maps;
        bool ok;
        if (args.a_codes) {
            cuuint64_t dims[2] = {(args.k + 1) / 2, args.m}, strides[1] = {args.a_codes_stride};
            cuuint32_t box[2] = {128, kBM}, steps[2] = {1, 1};
            ok = get_encode_tiled()(&maps.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(args.a_codes), dims, strides, box, steps,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
        } else {
            ok = line_map(maps.a, dev.a_codes, a_chunks * kBM, kBM);
        }
        ok = ok && line_map(maps.b, dev.b_codes, b_chunks * kBM, kBM);
        if (!ok) return cudaErrorInvalidValue;
        const uint64_t tiles = (args.tiles ? args.max_tiles : dev.tiles_m) * (uint64_t)dev.tiles_n;
        return args.c_bf16 ? launch_pair<true>(maps, dev, tiles, stream) : launch_pair<false>(maps, dev, tiles, stream);
    }
    if (args.a_codes) return cudaErrorInvalidValue;
    dev.tiles_m = (uint32_t)((args.m + kBM - 1) / kBM);
    // Narrower tiles while the wide ones are fewer than the SMs: a product with few rows is bound by the packed matrix's bytes, and every SM
    // that streams some of it counts. Sums run over the depth in the same order whatever the tile.
    const uint64_t row_tiles = args.tiles ? args.max_tiles : dev.tiles_m;
    int bn = 128;
    if (row_tiles * ((args.n + bn - 1) / bn) * 4 < (uint64_t)usable_sms() * 3) bn = 64;
    dev.tiles_n = (uint32_t)((args.n + bn - 1) / bn);
    const uint64_t tiles = row_tiles * dev.tiles_n;
    if (tiles > 0x7fffffffull) return cudaErrorInvalidValue;
    if (args.x) return launch_by_width<16, true>(bn, args.c_bf16, dev, tiles, stream);
    if (!args.tiles && args.m <= 16) return launch_by_width<16, false>(bn, args.c_bf16, dev, tiles, stream);
    return launch_by_width<128, false>(bn, args.c_bf16, dev, tiles, stream);
}

} // namespace nkb
