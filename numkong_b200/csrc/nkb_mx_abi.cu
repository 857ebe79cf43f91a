// Host side of the microscaled 4-bit and routing entry points: argument checks, operands that live in host memory, workspaces.
//
// A call whose operands are all device memory only enqueues kernels. Operands in host memory are copied to device buffers of
// the call's own, and the call returns when the results are back. Workspaces are the caller's where one is given, so that calls
// on several streams and captured graphs need not share one; without it the calling thread's staging memory is used.
#include <cstdio>
#include <cstring>

#include "../../include/numkong_b200.h"
#include "nkb_host.h"
#include "nkb_mx.h"

namespace nkb {
namespace {

bool float_type(uint32_t t) { return t == kF32 || t == kF16 || t == kBF16; }

// Device views of one call's operands.
class Operands {
public:
    explicit Operands(cudaStream_t stream) : stream_(stream) { cudaGetDevice(&device_); }
    Operands(const Operands &) = delete;
    ~Operands() {
        if (!on_host()) return;
        cudaStreamSynchronize(stream_);
        for (int i = 0; i < owned_count_; ++i) cudaFree(owned_[i]);
        cudaGetLastError();
    }
    bool on_host() const { return owned_count_ != 0; }

    // An input of `rows` rows of `row_bytes`, `stride` apart; a host matrix is uploaded with its rows packed 16-byte aligned. `stride` becomes
    // that of the device view, so it has to be the caller's copy of what it was given: a failed call fills the given rows.
    const uint8_t *in(const void *p, uint64_t rows, uint64_t row_bytes, uint64_t &stride) {
        if (!place(p)) return nullptr;
        if (on_device_) return static_cast<const uint8_t *>(p);
        const uint64_t pitch = round_up(row_bytes, 16);
        uint8_t *d = allocate(rows * pitch);
        if (!d || !cuda_ok(cudaMemcpy2DAsync(d, pitch, p, stride < row_bytes ? row_bytes : stride, row_bytes, rows, cudaMemcpyHostToDevice, stream_), "upload of operand")) return nullptr;
        stride = pitch;
        return d;
    }
    uint8_t *out(void *p, uint64_t rows, uint64_t row_bytes, uint64_t &stride) {
        if (!place(p)) return nullptr;
        if (on_device_) return static_cast<uint8_t *>(p);
        const uint64_t pitch = round_up(row_bytes, 16);
        uint8_t *d = allocate(rows * pitch);
        if (!d) return nullptr;
        results_[result_count_++] = {p, d, rows, row_bytes, stride < row_bytes ? row_bytes : stride, pitch};
        stride = pitch;
        return d;
    }
    // Where a packed blob or a workspace lives; false when it may not be used here.
    bool look(const void *p, MemKind &kind) {
        if (!place(p)) return false;
        kind = on_device_ ? kMemDevice : kMemHost;
        return true;
    }
    // Vectors: one dense row.
    const uint8_t *in(const void *p, uint64_t bytes) { uint64_t s = bytes; return in(p, 1, bytes, s); }
    uint8_t *out(void *p, uint64_t bytes) { uint64_t s = bytes; return out(p, 1, bytes, s); }

    // Copies host results back and waits for them, when the call had a host operand.
    bool finish(const char *what) {
        for (int i = 0; i < result_count_; ++i) {
            const Result &r = results_[i];
            if (!cuda_ok(cudaMemcpy2DAsync(r.host, r.stride, r.device, r.pitch, r.row_bytes, r.rows, cudaMemcpyDeviceToHost, stream_), "download of result")) return false;
        }
        if (!on_host()) return true;
        if (!cuda_ok(cudaStreamSynchronize(stream_), what)) return false;
        const uint32_t w = read_device_error();
        if (w) {
            char buf[64];
            std::snprintf(buf, sizeof buf, "0x%08x", w);
            set_error("a pipeline wait inside the GEMM kernel gave up (error word %s)", buf);
            return false;
        }
        return true;
    }

private:
    struct Result { void *host; uint8_t *device; uint64_t rows, row_bytes, stride, pitch; };
    bool place(const void *p) {
        cudaPointerAttributes attr;
        if (cudaPointerGetAttributes(&attr, p) != cudaSuccess) { cudaGetLastError(); on_device_ = false; return true; }
        on_device_ = attr.type == cudaMemoryTypeDevice || attr.type == cudaMemoryTypeManaged;
        if (attr.type == cudaMemoryTypeDevice && attr.device != device_) {
            set_error("an operand lives on another GPU than the calling thread's current one%s", "");
            return false;
        }
        return true;
    }
    uint8_t *allocate(uint64_t bytes) {
        void *p = nullptr;
        if (!cuda_ok(cudaMalloc(&p, bytes ? bytes : 16), "cudaMalloc(operand)")) return nullptr;
        owned_[owned_count_++] = p;
        return static_cast<uint8_t *>(p);
    }
    cudaStream_t stream_;
    int device_ = 0;
    bool on_device_ = false;
    void *owned_[6];  // no call has more operands, nor more than two results
    Result results_[2];
    int owned_count_ = 0, result_count_ = 0;
};

void refuse(const char *why) { set_error("%s", why); }

constexpr uint64_t kMostRows = 0x7fffff00ull;  // indices inside the kernels are 32 bits wide

bool on_another_gpu(const void *p) {
    cudaPointerAttributes attr;
    int device = 0;
    cudaGetDevice(&device);
    if (cudaPointerGetAttributes(&attr, p) != cudaSuccess) { cudaGetLastError(); return false; }
    return attr.type == cudaMemoryTypeDevice && attr.device != device;
}

// What an output holds after a refused or failed call: 0xFF bytes (NaN scales and cells, ids of -1), no more of them than the caller's
// sizes and stride span. Sizes that no kernel takes are not believed, another GPU's memory is left alone.
void spoil(void *out, uint64_t rows, uint64_t row_bytes, uint64_t stride) {
    if (!out || rows == 0 || rows > kMostRows || row_bytes > 4 * kMostRows || on_another_gpu(out)) return;
    if (stride < row_bytes) fill_error_output(out, classify(out), 1, (rows - 1) * stride + row_bytes, (rows - 1) * stride + row_bytes);
    else fill_error_output(out, classify(out), rows, row_bytes, stride);
}

uint64_t chunk_bytes(uint64_t rows, uint64_t depth) { return mx_geometry(1, rows, depth).row_blocks * mx_geometry(1, rows, depth).depth_blocks * kMxChunkBytes; }

uint8_t *workspace_or_scratch(Operands &ops, void *workspace, uint64_t bytes) {
    if (!workspace) {
        // Replays of two graphs may run at the same time, and a graph outlives what the thread's staging memory is next used for.
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        if (!cuda_ok(cudaStreamIsCapturing(current_stream(), &capture), "cudaStreamIsCapturing")) return nullptr;
        if (capture != cudaStreamCaptureStatusNone) {
            refuse("a call that is captured into a graph needs a workspace of its own");
            return nullptr;
        }
        return static_cast<uint8_t *>(scratch(kSlotA, bytes));
    }
    MemKind kind;
    if (!ops.look(workspace, kind)) return nullptr;
    if (kind != kMemDevice || (reinterpret_cast<uintptr_t>(workspace) & 255u)) {
        refuse("the workspace must be device memory on a 256-byte boundary");
        return nullptr;
    }
    return static_cast<uint8_t *>(workspace);
}

struct ExpertsLayout {
    uint32_t tile_rows;
    uint64_t max_tiles, tiles, count, dest, chunks, sums, total;
};
ExpertsLayout experts_layout(uint64_t slots, uint64_t experts, uint64_t width, uint64_t depth, bool weighted) {
    ExpertsLayout l;
    // CTA pairs on 256 rows fetch less per product but leave more of a tile empty at each expert's end: from 192 rows an expert on.
    // 32 experts of 2048 x 2048, 128 / 192 / 256 / 512 rows each: 33.3 / 39.1 / 46.6 / 74.7 us with 128 rows, 35.1 / 39.0 / 45.1 / 68.0 with 256.
    l.tile_rows = slots >= 192 * experts ? 256 : 128;
    l.max_tiles = slots / l.tile_rows + (slots < experts ? slots : experts);
    l.tiles = 0;
    l.count = round_up(l.max_tiles * sizeof(MxRowTile), 256);
    l.dest = l.count + 256;
    l.chunks = round_up(l.dest + l.max_tiles * l.tile_rows * 4, 256);
    l.sums = round_up(l.chunks + chunk_bytes(l.max_tiles * l.tile_rows, depth), 256);
    l.total = l.sums + (weighted ? slots * width * 4 : 0);
    return l;
}

// A . B^T with A given as codes and scales or, unless `coded`, as floats that are quantised on their way.
void product(bool coded, const void *a, uint32_t a_type, uint64_t a_stride, const void *codes, uint64_t codes_stride, const void *scales, uint64_t scales_stride,
             const void *packed, void *c, uint32_t c_type, uint64_t m, uint64_t n, uint64_t k, uint64_t c_stride, void *workspace) {
    clear_error();
    if (m == 0 || n == 0) return;
    if (m > kMostRows || n > kMostRows || k > kMostRows) return refuse("mxfp4 product: a size does not fit 31 bits");
    const uint32_t cell = dtype_bytes(c_type);
    const uint64_t row_bytes = n * cell;
    auto fail = [&]() { spoil(c, m, row_bytes, c_stride); };
    if ((c_type != kF32 && c_type != kBF16) || (!coded && !float_type(a_type))) { refuse("mxfp4 product: unsupported element type"); return fail(); }
    if (!packed || !c || (k && !(coded ? codes && scales : a != nullptr))) { refuse("mxfp4 product: null pointer"); return fail(); }
    if ((m > 1 && c_stride < row_bytes) || (reinterpret_cast<uintptr_t>(c) | (m > 1 ? c_stride : 0)) % cell) { refuse("mxfp4 product: rows of the result overlap or are not aligned to its cells"); return fail(); }
    const uint64_t kblocks = (k + kMxBlock - 1) / kMxBlock;
    if (m > 1 && (coded ? codes_stride < (k + 1) / 2 || scales_stride < kblocks : a_stride < k * dtype_bytes(a_type))) { refuse("mxfp4 product: rows of A overlap"); return fail(); }
    if (!coded && (reinterpret_cast<uintptr_t>(a) | (m > 1 ? a_stride : 0)) % dtype_bytes(a_type)) { refuse("mxfp4 product: values of A are not aligned to their type"); return fail(); }
    if (m == 1) c_stride = round_up(row_bytes, 16);  // whatever it was: nothing lies that far
    cudaStream_t stream = current_stream();
    Operands ops(stream);
    const MxGeometry g = mx_geometry(1, n, k);
    MemKind packed_kind;
    if (!ops.look(packed, packed_kind)) return fail();
    const uint8_t *blob = resident_blob_of_size(packed, packed_kind, kMagicMx, kMxfp4, n, k, g.total_bytes, nullptr);
    unsigned int *err = blob ? device_error_word() : nullptr;
    if (!err) { if (blob) refuse("could not allocate the device error word"); return fail(); }
    uint64_t c_pitch = c_stride;
    uint8_t *c_dev = ops.out(c, m, row_bytes, c_pitch);
    bool ok = c_dev != nullptr;
    if (ok && k == 0) ok = cuda_ok(cudaMemset2DAsync(c_dev, c_pitch, 0, row_bytes, m, stream), "clear result");
    else if (ok) {
        const uint8_t *ad = nullptr;
        if (!coded) {
            ad = ops.in(a, m, k * dtype_bytes(a_type), a_stride);
            ok = ad != nullptr;
        }
        // A that the product quantises itself is read until its last CTA is through, so C may not lie over it.
        const uint64_t a_span = (m - 1) * a_stride + k * dtype_bytes(a_type), c_span = (m - 1) * c_pitch + row_bytes;
        const bool inside = !coded && gemm_mx_quantises(m) && !(c_dev < ad + a_span && ad < c_dev + c_span);
        uint8_t *chunks = !ok || inside ? nullptr : workspace_or_scratch(ops, workspace, chunk_bytes(m, k));
        ok = ok && (inside || chunks);
        bool rows_in_place = false;
        const uint8_t *cd = nullptr;
        if (ok && coded) {
            cd = ops.in(codes, m, (k + 1) / 2, codes_stride);
            const uint8_t *sd = cd ? ops.in(scales, m, kblocks, scales_stride) : nullptr;
            if (m == 1) codes_stride = round_up((k + 1) / 2, 16);
            rows_in_place = sd && gemm_mx_reads_rows(m, n, k) && ((reinterpret_cast<uintptr_t>(cd) | codes_stride) & 15u) == 0;
            if (rows_in_place) ok = cuda_ok(launch_mx_tile_scales(sd, scales_stride, m, k, chunks, stream), "scale tile kernel");
            else ok = sd && cuda_ok(launch_mx_tile(cd, codes_stride, sd, scales_stride, 1, m, k, false, chunks, stream), "tile kernel");
        } else if (ok && !inside) {
            ok = cuda_ok(launch_mx_quantise_tiled(a_type, ad, k, m > 1 ? a_stride : 0, m, nullptr, nullptr, 0, 1, chunks, stream), "quantise kernel");
        }
        if (ok) {
            MxGemmArgs args;
            args.a_chunks = chunks; args.b_chunks = blob + g.payload_offset;
            if (inside) { args.x = ad; args.x_stride = m > 1 ? a_stride : 0; args.x_type = a_type; }
            if (rows_in_place) { args.a_codes = cd; args.a_codes_stride = codes_stride; }
            args.c = c_dev; args.c_stride = c_pitch; args.c_bf16 = c_type == kBF16;
            args.m = m; args.n = n; args.k = k; args.error_word = err;
            ok = cuda_ok(launch_gemm_mx(args, stream), "mxfp4 GEMM kernel");
            g_launches += inside ? 1 : 2;
        }
    }
    if (ok && packed_kind == kMemHost && !ops.on_host()) ok = cuda_ok(cudaStreamSynchronize(stream), "mxfp4 product");
    if (!ok || !ops.finish("mxfp4 product")) fail();
}

} // namespace
} // namespace nkb

using namespace nkb;

extern "C" {

NKB_API void nkb_mx_quantise(void const *x, uint32_t x_type, nk_size_t rows, nk_size_t depth, nk_size_t x_stride, void *codes,
                             nk_size_t codes_stride, void *scales, nk_size_t scales_stride) {
    clear_error();
    if (rows == 0 || depth == 0) return;
    if (rows > kMostRows || depth > kMostRows) return refuse("mx_quantise: a size does not fit 31 bits");
    const uint64_t code_bytes = (depth + 1) / 2, blocks = (depth + kMxBlock - 1) / kMxBlock;
    auto fail = [&]() {
        spoil(codes, rows, code_bytes, codes_stride);
        spoil(scales, rows, blocks, scales_stride);
    };
    if (!float_type(x_type) || !x || !codes || !scales) { refuse("mx_quantise: unsupported element type or null pointer"); return fail(); }
    if (rows > 1 && (x_stride < depth * dtype_bytes(x_type) || codes_stride < code_bytes || scales_stride < blocks)) { refuse("mx_quantise: rows overlap"); return fail(); }
    if ((reinterpret_cast<uintptr_t>(x) | (rows > 1 ? x_stride : 0)) % dtype_bytes(x_type)) { refuse("mx_quantise: values are not aligned to their type"); return fail(); }
    cudaStream_t stream = current_stream();
    Operands ops(stream);
    const uint8_t *xd = ops.in(x, rows, depth * dtype_bytes(x_type), x_stride);
    uint64_t codes_pitch = codes_stride, scales_pitch = scales_stride;
    uint8_t *cd = xd ? ops.out(codes, rows, code_bytes, codes_pitch) : nullptr, *sd = cd ? ops.out(scales, rows, blocks, scales_pitch) : nullptr;
    const bool ok = sd && cuda_ok(launch_mx_quantise(x_type, xd, rows, depth, x_stride, cd, codes_pitch, sd, scales_pitch, stream), "quantise kernel");
    g_launches++;
    if (!ok || !ops.finish("mx_quantise")) fail();
}

NKB_API void nkb_mx_dequantise(void const *codes, nk_size_t codes_stride, void const *scales, nk_size_t scales_stride, nk_size_t rows,
                               nk_size_t depth, void *x, uint32_t x_type, nk_size_t x_stride) {
    clear_error();
    if (rows == 0 || depth == 0) return;
    if (rows > kMostRows || depth > kMostRows) return refuse("mx_dequantise: a size does not fit 31 bits");
    const uint64_t code_bytes = (depth + 1) / 2, blocks = (depth + kMxBlock - 1) / kMxBlock;
    const uint64_t row_bytes = depth * dtype_bytes(x_type);
    auto fail = [&]() { spoil(x, rows, row_bytes, x_stride); };
    if (!float_type(x_type)) { refuse("mx_dequantise: unsupported element type"); return fail(); }
    if (!x || !codes || !scales) { refuse("mx_dequantise: null pointer"); return fail(); }
    if (rows > 1 && (x_stride < row_bytes || codes_stride < code_bytes || scales_stride < blocks)) { refuse("mx_dequantise: rows overlap"); return fail(); }
    if ((reinterpret_cast<uintptr_t>(x) | (rows > 1 ? x_stride : 0)) % dtype_bytes(x_type)) { refuse("mx_dequantise: values are not aligned to their type"); return fail(); }
    cudaStream_t stream = current_stream();
    Operands ops(stream);
    const uint8_t *cd = ops.in(codes, rows, code_bytes, codes_stride), *sd = cd ? ops.in(scales, rows, blocks, scales_stride) : nullptr;
    uint64_t x_pitch = x_stride;
    uint8_t *xd = sd ? ops.out(x, rows, row_bytes, x_pitch) : nullptr;
    const bool ok = xd && cuda_ok(launch_mx_dequantise(x_type, cd, codes_stride, sd, scales_stride, rows, depth, xd, x_pitch, stream), "dequantise kernel");
    g_launches++;
    if (!ok || !ops.finish("mx_dequantise")) fail();
}

NKB_API nk_size_t nkb_dots_packed_size_mxfp4(nk_size_t groups, nk_size_t width, nk_size_t depth) {
    return mx_geometry(groups, width, depth).total_bytes;
}

NKB_API void nkb_dots_pack_mxfp4(void const *codes, nk_size_t codes_stride, void const *scales, nk_size_t scales_stride, nk_size_t groups,
                                 nk_size_t width, nk_size_t depth, void *packed) {
    clear_error();
    if (!packed) return refuse("mxfp4 pack: null output");
    if (groups > kMostRows || width > kMostRows || depth > kMostRows || mx_geometry(groups, width, depth).row_blocks * kChunkRows > kMostRows) return refuse("mxfp4 pack: a size does not fit 31 bits");
    const MxGeometry g = mx_geometry(groups, width, depth);
    const uint64_t rows = groups * width, code_bytes = (depth + 1) / 2, blocks = (depth + kMxBlock - 1) / kMxBlock;
    const MemKind out_kind = classify(packed);
    auto fail = [&]() { if (!on_another_gpu(packed)) fill_error_output(packed, out_kind, 1, g.total_bytes, g.total_bytes); };
    if (rows && depth && (!codes || !scales)) { refuse("mxfp4 pack: null input"); return fail(); }
    if (rows > 1 && (codes_stride < code_bytes || scales_stride < blocks)) { refuse("mxfp4 pack: rows overlap"); return fail(); }
    if (out_kind == kMemDevice && (reinterpret_cast<uintptr_t>(packed) & 15u)) { refuse("pack: device output must be 16-byte aligned"); return fail(); }
    PackedHeader h;
    std::memset(&h, 0, sizeof h);
    h.magic = kMagicMx; h.dtype = kMxfp4; h.element_bytes = 1; h.norm_bytes = 0;
    h.rows = rows; h.depth = depth; h.rows_padded = g.row_blocks * kChunkRows; h.depth_padded_bytes = g.depth_blocks * 128;
    h.payload_offset = g.payload_offset; h.norms_offset = g.total_bytes; h.total_bytes = g.total_bytes;
    h.nonce = fresh_nonce(); h.reserved[0] = groups;
    cudaStream_t stream = current_stream();
    Operands ops(stream);
    MemKind looked;
    if (!ops.look(packed, looked)) return fail();
    uint8_t *blob = static_cast<uint8_t *>(packed);
    if (out_kind == kMemHost) {
        void *d = nullptr;
        if (!cuda_ok(cudaMalloc(&d, g.total_bytes), "cudaMalloc(packed blob)")) return fail();
        blob = static_cast<uint8_t *>(d);
    }
    bool ok = true;
    if (rows && depth) {
        const uint8_t *cd = ops.in(codes, rows, code_bytes, codes_stride), *sd = cd ? ops.in(scales, rows, blocks, scales_stride) : nullptr;
        ok = sd && cuda_ok(launch_mx_tile(cd, codes_stride, sd, scales_stride, groups, width, depth, true, blob + g.payload_offset, stream), "tile kernel");
    }
    ok = ok && cuda_ok(launch_write_header(blob, h, stream), "header kernel");
    g_launches += 2;
    if (out_kind == kMemHost) {
        ok = ok && cuda_ok(cudaMemcpyAsync(packed, blob, g.total_bytes, cudaMemcpyDeviceToHost, stream), "download of packed blob") &&
             cuda_ok(cudaStreamSynchronize(stream), "mxfp4 pack");
        if (ok) remember_blob(h.nonce, g.total_bytes, blob);
        else cudaFree(blob);
    }
    if (!ok || !ops.finish("mxfp4 pack")) fail();
}

NKB_API nk_size_t nkb_dots_workspace_mxfp4(nk_size_t height, nk_size_t depth) { return chunk_bytes(height, depth); }

NKB_API void nkb_dots_packed_mxfp4(void const *codes, nk_size_t codes_stride, void const *scales, nk_size_t scales_stride, void const *b_packed,
                                   void *c, uint32_t c_type, nk_size_t height, nk_size_t width, nk_size_t depth, nk_size_t c_stride, void *workspace) {
    product(true, nullptr, 0, 0, codes, codes_stride, scales, scales_stride, b_packed, c, c_type, height, width, depth, c_stride, workspace);
}

NKB_API void nkb_dots_packed_quantised_mxfp4(void const *a, uint32_t a_type, nk_size_t a_stride, void const *b_packed, void *c, uint32_t c_type,
                                             nk_size_t height, nk_size_t width, nk_size_t depth, nk_size_t c_stride, void *workspace) {
    product(false, a, a_type, a_stride, nullptr, 0, nullptr, 0, b_packed, c, c_type, height, width, depth, c_stride, workspace);
}

NKB_API void nkb_route(void const *logits, uint32_t type, nk_size_t tokens, nk_size_t experts, nk_size_t logits_stride, float const *bias,
                       uint32_t score, nk_size_t groups, nk_size_t top_groups, nk_size_t top, int renormalise, float scale, float *weights, int32_t *ids) {
    clear_error();
    if (tokens == 0) return;
    if (tokens > kMostRows) return refuse("route: the tokens do not fit 31 bits");
    auto fail = [&]() {
        spoil(weights, tokens, top * 4, top * 4);
        spoil(ids, tokens, top * 4, top * 4);
    };
    if (top == 0 || top > kRouteMaxTop || experts == 0 || experts > kRouteMaxExperts || top > experts) { refuse("route: 1 to 32 choices of 1 to 1024 experts"); return top <= kRouteMaxTop ? fail() : void(); }
    if (!float_type(type) || score > 1 || !logits || !weights || !ids) { refuse("route: unsupported element type or score, or null pointer"); return fail(); }
    if (groups == 0 || groups > kRouteMaxGroups || experts % groups || top_groups == 0 || top_groups > groups) { refuse("route: up to 32 groups of equal size, of which at least one and at most all are open"); return fail(); }
    if (tokens > 1 && logits_stride < experts * dtype_bytes(type)) { refuse("route: rows overlap"); return fail(); }
    if ((reinterpret_cast<uintptr_t>(logits) | (tokens > 1 ? logits_stride : 0)) % dtype_bytes(type) || (reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(ids)) % 4) { refuse("route: operands are not aligned to their elements"); return fail(); }
    cudaStream_t stream = current_stream();
    Operands ops(stream);
    RouteArgs a;
    uint64_t stride = logits_stride;
    a.logits = ops.in(logits, tokens, experts * dtype_bytes(type), stride);
    a.bias = a.logits && bias ? reinterpret_cast<const float *>(ops.in(bias, experts * 4)) : nullptr;
    float *w = a.logits && (!bias || a.bias) ? reinterpret_cast<float *>(ops.out(weights, tokens * top * 4)) : nullptr;
    int32_t *i = w ? reinterpret_cast<int32_t *>(ops.out(ids, tokens * top * 4)) : nullptr;
    a.type = type; a.tokens = tokens; a.logits_stride = stride;
    a.experts = (uint32_t)experts; a.groups = (uint32_t)groups; a.top_groups = (uint32_t)top_groups; a.top = (uint32_t)top;
    a.sigmoid = score == 1; a.renormalise = renormalise != 0; a.scale = scale;
    const bool ok = i && cuda_ok(launch_route(a, w, i, stream), "route kernel");
    g_launches++;
    if (!ok || !ops.finish("route")) fail();
}

NKB_API void nkb_route_gradient(float const *weights_grad, int32_t const *ids, void const *logits, uint32_t type, nk_size_t tokens, nk_size_t experts,
                                nk_size_t logits_stride, uint32_t score, nk_size_t top, int renormalise, float scale, float *logits_grad) {
    clear_error();
    if (tokens == 0) return;
    if (tokens > kMostRows) return refuse("route_gradient: the tokens do not fit 31 bits");
    auto fail = [&]() { if (experts <= kRouteMaxExperts) spoil(logits_grad, tokens, experts * 4, experts * 4); };
    if (top == 0 || top > kRouteMaxTop || experts == 0 || experts > kRouteMaxExperts) { refuse("route_gradient: 1 to 32 choices of 1 to 1024 experts"); return fail(); }
    if (!float_type(type) || score > 1 || !logits || !weights_grad || !ids || !logits_grad) { refuse("route_gradient: unsupported element type or score, or null pointer"); return fail(); }
    if (tokens > 1 && logits_stride < experts * dtype_bytes(type)) { refuse("route_gradient: rows overlap"); return fail(); }
    if ((reinterpret_cast<uintptr_t>(logits) | (tokens > 1 ? logits_stride : 0)) % dtype_bytes(type) || (reinterpret_cast<uintptr_t>(weights_grad) | reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(logits_grad)) % 4) { refuse("route_gradient: operands are not aligned to their elements"); return fail(); }
    cudaStream_t stream = current_stream();
    Operands ops(stream);
    RouteArgs a;
    uint64_t stride = logits_stride;
    a.logits = ops.in(logits, tokens, experts * dtype_bytes(type), stride);
    const float *w = a.logits ? reinterpret_cast<const float *>(ops.in(weights_grad, tokens * top * 4)) : nullptr;
    const int32_t *i = w ? reinterpret_cast<const int32_t *>(ops.in(ids, tokens * top * 4)) : nullptr;
    float *g = i ? reinterpret_cast<float *>(ops.out(logits_grad, tokens * experts * 4)) : nullptr;
    a.type = type; a.tokens = tokens; a.logits_stride = stride; a.bias = nullptr;
    a.experts = (uint32_t)experts; a.groups = 1; a.top_groups = 1; a.top = (uint32_t)top;
    a.sigmoid = score == 1; a.renormalise = renormalise != 0; a.scale = scale;
    const bool ok = g && cuda_ok(launch_route_gradient(a, w, i, g, stream), "route gradient kernel");
    g_launches++;
    if (!ok || !ops.finish("route_gradient")) fail();
}

NKB_API nk_size_t nkb_experts_workspace_mxfp4(nk_size_t tokens, nk_size_t top, nk_size_t experts, nk_size_t width, nk_size_t depth, int weighted) {
    return experts_layout(tokens * top, experts, width, depth, weighted != 0).total;
}

NKB_API void nkb_experts_packed_mxfp4(void const *x, uint32_t x_type, nk_size_t x_stride, int per_slot, int32_t const *ids, nk_size_t tokens, nk_size_t top,
                                      void const *b_packed, nk_size_t experts, nk_size_t width, nk_size_t depth, float const *weights, void *out,
                                      uint32_t out_type, nk_size_t out_stride, void *workspace) {
    clear_error();
    if (tokens == 0 || width == 0) return;
    if (tokens > kMostRows || top == 0 || top > 1024 || tokens * top > kMostRows / 2 || width > kMostRows || depth > kMostRows) return refuse("experts: 1 to 1024 choices, and sizes that fit 31 bits");
    const uint64_t slots = tokens * top, rows = weights ? tokens : slots, x_rows = per_slot ? slots : tokens;
    const uint32_t cell = dtype_bytes(out_type);
    const uint64_t row_bytes = width * cell;
    auto fail = [&]() { spoil(out, rows, row_bytes, out_stride); };
    if (!float_type(x_type) || (out_type != kF32 && out_type != kBF16)) { refuse("experts: unsupported element type"); return fail(); }
    if (!ids || !b_packed || !out || (depth && !x)) { refuse("experts: null pointer"); return fail(); }
    if (experts == 0 || experts > kRouteMaxExperts) { refuse("experts: 1 to 1024 experts"); return fail(); }
    if ((x_rows > 1 && x_stride < depth * dtype_bytes(x_type)) || (rows > 1 && out_stride < row_bytes)) { refuse("experts: rows overlap"); return fail(); }
    if ((reinterpret_cast<uintptr_t>(x) | (x_rows > 1 ? x_stride : 0)) % dtype_bytes(x_type) || (reinterpret_cast<uintptr_t>(out) | (rows > 1 ? out_stride : 0)) % cell || (reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights)) % 4) { refuse("experts: operands are not aligned to their elements"); return fail(); }
    if (rows == 1) out_stride = round_up(row_bytes, 16);
    cudaStream_t stream = current_stream();
    Operands ops(stream);
    const MxGeometry g = mx_geometry(experts, width, depth);
    MemKind packed_kind;
    if (!ops.look(b_packed, packed_kind)) return fail();
    const uint8_t *blob = resident_blob_of_size(b_packed, packed_kind, kMagicMx, kMxfp4, experts * width, depth, g.total_bytes, nullptr);
    unsigned int *err = blob ? device_error_word() : nullptr;
    if (!err) { if (blob) refuse("could not allocate the device error word"); return fail(); }
    uint64_t out_pitch = out_stride;
    uint8_t *dst = ops.out(out, rows, row_bytes, out_pitch);
    bool ok = dst != nullptr;
    if (ok && depth == 0) ok = cuda_ok(cudaMemset2DAsync(dst, out_pitch, 0, row_bytes, rows, stream), "clear result");
    else if (ok) {
        const ExpertsLayout l = experts_layout(slots, experts, width, depth, weights != nullptr);
        uint8_t *ws = workspace_or_scratch(ops, workspace, l.total);
        const int32_t *id = ws ? reinterpret_cast<const int32_t *>(ops.in(ids, slots * 4)) : nullptr;
        const uint8_t *xd = id ? ops.in(x, x_rows, depth * dtype_bytes(x_type), x_stride) : nullptr;
        const float *wd = xd && weights ? reinterpret_cast<const float *>(ops.in(weights, slots * 4)) : nullptr;
        ok = xd && (!weights || wd);
        if (ok) {
            MxRowTile *tiles = reinterpret_cast<MxRowTile *>(ws + l.tiles);
            int32_t *count = reinterpret_cast<int32_t *>(ws + l.count), *dest = reinterpret_cast<int32_t *>(ws + l.dest);
            float *sums = reinterpret_cast<float *>(ws + l.sums);
            MxGemmArgs args;
            args.a_chunks = ws + l.chunks; args.b_chunks = blob + g.payload_offset;
            args.c = weights ? static_cast<void *>(sums) : dst; args.c_stride = weights ? width * 4 : out_pitch;
            args.c_bf16 = !weights && out_type == kBF16;
            args.m = slots; args.n = width; args.k = depth;
            args.tiles = tiles; args.tile_count = count; args.row_dest = dest; args.max_tiles = l.max_tiles; args.tile_rows = l.tile_rows; args.groups = experts; args.error_word = err;
            const uint32_t divide = per_slot ? 1u : (uint32_t)top, n = (uint32_t)experts;
            const uint64_t stride = x_rows > 1 ? x_stride : 0;
            args.tiles_fresh = slots <= kFewSlots;
            if (args.tiles_fresh)
                ok = cuda_ok(launch_order_and_quantise(x_type, xd, depth, stride, id, (uint32_t)slots, n, divide, l.tile_rows, l.max_tiles, tiles, count, dest, weights ? nullptr : dst,
                                                       row_bytes, out_pitch, ws + l.chunks, stream), "order and quantise kernel");
            else
                ok = cuda_ok(launch_expert_order(id, slots, n, tiles, count, dest, l.max_tiles, l.tile_rows, stream), "expert order kernel") &&
                     cuda_ok(launch_mx_quantise_tiled(x_type, xd, depth, stride, l.max_tiles * l.tile_rows, dest, count, l.tile_rows, divide, ws + l.chunks, stream), "quantise kernel");
            ok = ok && cuda_ok(launch_gemm_mx(args, stream), "grouped mxfp4 GEMM kernel");
            if (ok && weights) ok = cuda_ok(launch_combine(sums, wd, id, tokens, (uint32_t)top, n, width, dst, out_type == kBF16, out_pitch, stream), "combine kernel");
            else if (ok && !args.tiles_fresh) ok = cuda_ok(launch_zero_unrouted(id, slots, n, dst, row_bytes, out_pitch, stream), "zero kernel");
            g_launches += !args.tiles_fresh ? 4 : weights ? 3 : 2;
        }
    }
    if (ok && packed_kind == kMemHost && !ops.on_host()) ok = cuda_ok(cudaStreamSynchronize(stream), "experts");
    if (!ok || !ops.finish("experts")) fail();
}

} // extern "C"
