// Microscaled 4-bit floats (MXFP4): the tile layout the tensor cores read, the packed blob built from it, and the launchers
// of the conversions, the product and the expert order.
//
// A value is an e2m1 code (sign, two exponent bits, one mantissa bit: 0 .5 1 1.5 2 3 4 6) times a scale 2^(s - 127) that 32
// consecutive values of a row share; s = 255 is NaN. Row-major form, as callers hold it: two codes per byte, the even value in
// the low half, ceil(depth / 2) bytes of codes and ceil(depth / 32) scale bytes per row.
//
// Tile form: a chunk is 128 rows x 256 values. Its codes are 16 KiB, 128 bytes per row, in the 128-byte-swizzled K-major image
// tcgen05.mma reads (as in PackedHeader); its scales are two 512-byte tiles, one per 128 values of depth, each the image the MMA's
// scales take in TMEM: the four scales of row r at byte (r % 32) * 16 + (r / 32) * 4 (lane r % 32, column r / 32). All chunks' codes
// come first, then all chunks' scales, both ordered [row block][depth block], so that a CTA that stays on one row block reads two
// contiguous streams with nothing left to rearrange.
#pragma once
#include "nkb_internal.h"

namespace nkb {

constexpr uint32_t kMxfp4 = 1u << 28;            // this library's own code: the reference has no such type
constexpr uint32_t kMagicMx = 0x584D424Bu;       // "KBMX"
constexpr uint32_t kMxBlock = 32;                // values per scale
constexpr uint32_t kMxChunkValues = 256;         // values of depth per chunk
constexpr uint32_t kMxCodeBytes = kChunkBytes;   // 128 rows x 128 bytes
constexpr uint32_t kMxScaleBytes = 1024;
constexpr uint32_t kMxChunkBytes = kMxCodeBytes + kMxScaleBytes;

struct MxGeometry {
    uint64_t row_blocks;    // chunks of 128 rows, every group padded to whole chunks
    uint64_t depth_blocks;
    uint64_t payload_offset, total_bytes;
};
inline MxGeometry mx_geometry(uint64_t groups, uint64_t width, uint64_t depth) {
    MxGeometry g;
    g.row_blocks = groups * ((width + kChunkRows - 1) / kChunkRows);
    g.depth_blocks = (depth + kMxChunkValues - 1) / kMxChunkValues;
    g.payload_offset = kHeaderBytes;
    g.total_bytes = g.payload_offset + g.row_blocks * g.depth_blocks * kMxChunkBytes;
    return g;
}

// float rows -> row-major codes and scales.
cudaError_t launch_mx_quantise(uint32_t type, const void *x, uint64_t rows, uint64_t depth, uint64_t x_stride, void *codes,
                               uint64_t codes_stride, void *scales, uint64_t scales_stride, cudaStream_t stream);
// float rows -> tile form. Tiled row i is row i of x, or, with `row_dest`, row row_dest[i] / divide of x; entries below 0 leave
// their row as it is.
cudaError_t launch_mx_quantise_tiled(uint32_t type, const void *x, uint64_t depth, uint64_t x_stride, uint64_t tiled_rows,
                                     const int32_t *row_dest, const int32_t *tile_count, uint32_t tile_rows, uint32_t divide, void *chunks, cudaStream_t stream);
cudaError_t launch_mx_dequantise(uint32_t type, const void *codes, uint64_t codes_stride, const void *scales, uint64_t scales_stride,
                                 uint64_t rows, uint64_t depth, void *x, uint64_t x_stride, cudaStream_t stream);
// Row-major codes and scales -> tile form; `pad_rows`: rows behind the last one of every group are written too (zero codes, scale 1).
cudaError_t launch_mx_tile(const void *codes, uint64_t codes_stride, const void *scales, uint64_t scales_stride, uint64_t groups,
                           uint64_t width, uint64_t depth, bool pad_rows, void *chunks, cudaStream_t stream);

// Row-major scales -> scale tiles alone, 1024 bytes per 128 rows x 256 values.
cudaError_t launch_mx_tile_scales(const void *scales, uint64_t scales_stride, uint64_t rows, uint64_t depth, void *tiles, cudaStream_t stream);

// One row tile (128 or 256 rows of A in tile form, see MxGemmArgs::tile_rows) of a grouped product.
struct MxRowTile {
    int32_t group;  // packed matrix its rows multiply
    int32_t rows;   // valid rows, 1 .. 128 (256)
};
struct MxGemmArgs {
    const void *a_chunks;              // A in tile form; with `a_codes` set, its scale tiles alone
    const void *a_codes = nullptr;     // A's row-major codes (16-byte aligned, stride too), see gemm_mx_reads_rows
    uint64_t a_codes_stride = 0;
    const void *b_chunks;
    const void *x = nullptr;           // or float rows of A, quantised inside: see gemm_mx_quantises
    uint64_t x_stride = 0;
    uint32_t x_type = 0;
    void *c;
    uint64_t c_stride;
    bool c_bf16;                       // cells: bf16 (rounded to nearest even) or f32
    uint64_t m, n, k;                  // n: rows of one packed matrix
    const MxRowTile *tiles = nullptr;  // grouped product: row tiles, their count and the destination row of every tiled row
    const int32_t *tile_count = nullptr;
    const int32_t *row_dest = nullptr;
    uint64_t max_tiles = 0;            // row tiles there may be at most
    uint32_t tile_rows = 128;          // 256: CTA pairs
    bool tiles_fresh = false;          // the kernel just before writes the tiles, too
    uint64_t groups = 1;
    unsigned int *error_word = nullptr;
};
// Whether a product of this size reads A's codes from the caller's rows when they are aligned.
bool gemm_mx_reads_rows(uint64_t m, uint64_t n, uint64_t k);
// Whether a product with this many rows takes float rows as they are.
bool gemm_mx_quantises(uint64_t m);
cudaError_t launch_gemm_mx(const MxGemmArgs &args, cudaStream_t stream);

// ---- routing and the experts' products ----
struct RouteArgs {
    uint32_t type;                 // of the logits
    const void *logits;
    uint64_t tokens, logits_stride;
    uint32_t experts, groups, top_groups, top;
    bool sigmoid, renormalise;
    float scale;
    const float *bias;             // per expert, added for the selection only; may be null
};
constexpr uint32_t kRouteMaxExperts = 1024, kRouteMaxTop = 32, kRouteMaxGroups = 32;
cudaError_t launch_route(const RouteArgs &args, float *weights, int32_t *ids, cudaStream_t stream);
cudaError_t launch_route_gradient(const RouteArgs &args, const float *weights_grad, const int32_t *ids, float *logits_grad, cudaStream_t stream);

// Row tiles of at most `tile_rows` slots of one expert each. `slots` ids; those outside [0, experts) choose none.
cudaError_t launch_expert_order(const int32_t *ids, uint64_t slots, uint32_t experts, MxRowTile *tiles, int32_t *tile_count, int32_t *row_dest,
                                uint64_t max_tiles, uint32_t tile_rows, cudaStream_t stream);
// The same and the quantising of the slots' rows (x row slot / divide) in one launch, for at most kFewSlots slots; rows of `out`, where it is
// not null, whose slot chooses no expert are zeroed.
constexpr uint32_t kFewSlots = 256;
cudaError_t launch_order_and_quantise(uint32_t type, const void *x, uint64_t depth, uint64_t x_stride, const int32_t *ids, uint32_t slots, uint32_t experts, uint32_t divide,
                                      uint32_t tile_rows, uint64_t max_tiles, MxRowTile *tiles, int32_t *tile_count, int32_t *row_dest, void *out,
                                      uint64_t row_bytes, uint64_t out_stride, void *chunks, cudaStream_t stream);
// Zeros the rows of `out` whose slot chooses no expert.
cudaError_t launch_zero_unrouted(const int32_t *ids, uint64_t slots, uint32_t experts, void *out, uint64_t row_bytes, uint64_t out_stride, cudaStream_t stream);
// out[t] = sum over j of weights[t, j] * y[t * top + j], slots without an expert left out; f32 sums in order of j.
cudaError_t launch_combine(const float *y, const float *weights, const int32_t *ids, uint64_t tokens, uint32_t top, uint32_t experts, uint64_t width,
                           void *out, bool bf16, uint64_t out_stride, cudaStream_t stream);

} // namespace nkb
