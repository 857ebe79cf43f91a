// Routing of tokens to experts: scores from logits, selection, weights, and the gradient that trains the router.
//
//   score   s_e = softmax(l)_e or 1 / (1 + exp(-l_e))
//   choice  key_e = s_e + bias_e; with groups, a group is worth the sum of its two best keys and only the `top_groups` best
//           groups stay open; the `top` best open keys are chosen, best first, ties (of groups and of experts) to the lower index
//   weight  w_j = scale * s_{i_j}, or scale * s_{i_j} / sum over the chosen
//
// A logit of -infinity or NaN masks its expert: it has score 0 and is never chosen. A bias of -infinity or NaN only keeps its
// expert from being chosen. +infinity counts as the largest finite value. Slots that find no expert get id -1 and weight 0.
// Which of two near keys is the larger decides who is chosen, so keys are compared in 64 bits.
//
// Gradient, with p the chosen scores, g the incoming gradient times the scale and S their sum:
//   renormalised   d s_{i_j} = (g_j - sum_i g_i p_i / S) / S,   otherwise d s_{i_j} = g_j
//   softmax        d l_e = s_e (d s_e - sum_i d s_i s_i),       sigmoid d l_e = s_e (1 - s_e) d s_e
#include <cfloat>
#include "nkb_decode.cuh"
#include "nkb_mx.h"

namespace nkb {

namespace {

constexpr int kWarps = 4;

template <uint32_t kType>
__device__ __forceinline__ float load_logit(const uint8_t *row, uint32_t e) {
    float v;
    if constexpr (kType == kF32) v = reinterpret_cast<const float *>(row)[e];
    else v = decode_bits<kType>(reinterpret_cast<const uint16_t *>(row)[e]);
    return v == v ? fminf(v, FLT_MAX) : -INFINITY;  // NaN masks
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// The largest key of the warp and its index; the lower index where keys are equal.
__device__ __forceinline__ void warp_best(double &key, uint32_t &index) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const double k = __shfl_xor_sync(0xffffffffu, key, o);
        const uint32_t i = __shfl_xor_sync(0xffffffffu, index, o);
        if (k > key || (k == key && i < index)) { key = k; index = i; }
    }
}

struct RouteDev {
    const uint8_t *logits;
    uint64_t stride, tokens;
    uint32_t experts, groups, top_groups, top;
    float scale;
    const float *bias;
    bool sigmoid, renormalise;
};

__device__ __forceinline__ double log_sigmoid(double l) { return fmin(l, 0.0) - log1p(exp(-fabs(l))); }

template <uint32_t kType>
__global__ void __launch_bounds__(kWarps * 32) route_kernel(const RouteDev p, float *weights, int32_t *ids) {
    extern __shared__ double keys_all[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double *keys = keys_all + (size_t)warp * p.experts;
    for (uint64_t token = (uint64_t)blockIdx.x * kWarps + warp; token < p.tokens; token += (uint64_t)gridDim.x * kWarps) {
        const uint8_t *row = p.logits + token * p.stride;
        float top_logit = -INFINITY;
        for (uint32_t e = lane; e < p.experts; e += 32) top_logit = fmaxf(top_logit, load_logit<kType>(row, e));
        top_logit = warp_max(top_logit);
        double total = 0.0;
        if (!p.sigmoid) {
            for (uint32_t e = lane; e < p.experts; e += 32) {
                const float l = load_logit<kType>(row, e);
                if (l > -INFINITY) total += exp((double)l - top_logit);
            }
            total = warp_sum(total);
        }
        for (uint32_t e = lane; e < p.experts; e += 32) {
            const float l = load_logit<kType>(row, e);
            const float b = p.bias ? p.bias[e] : 0.0f;
            double key = -INFINITY;
            if (l > -INFINITY && b > -INFINITY)  // false for a NaN bias
                key = p.bias == nullptr && p.groups == 1 ? (double)l  // scores grow with their logits
                                        : (p.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : exp((double)l - top_logit) / total) + fminf(b, FLT_MAX);
            keys[e] = key;
        }
        __syncwarp();
        if (p.groups > 1) {
            const uint32_t size = p.experts / p.groups;
            double worth = -INFINITY;
            if ((uint32_t)lane < p.groups) {
                double first = -INFINITY, second = -INFINITY;
                for (uint32_t i = 0; i < size; ++i) {
                    const double k = keys[lane * size + i];
                    if (k > first) { second = first; first = k; }
                    else if (k > second) second = k;
                }
                worth = second > -INFINITY ? first + second : first;
            }
            bool open = false;
            double mine = worth;
            for (uint32_t g = 0; g < p.top_groups; ++g) {
                double best = mine;
                uint32_t who = lane;
                warp_best(best, who);
                if (best == -INFINITY) break;
                if (who == (uint32_t)lane) { open = true; mine = -INFINITY; }
            }
            if ((uint32_t)lane < p.groups && !open)
                for (uint32_t i = 0; i < size; ++i) keys[lane * size + i] = -INFINITY;
            __syncwarp();
        }
        int32_t chosen = -1;  // lane j: the expert of slot j
        for (uint32_t j = 0; j < p.top; ++j) {
            double best = -INFINITY;
            uint32_t who = 0xffffffffu;
            for (uint32_t e = lane; e < p.experts; e += 32)
                if (keys[e] > best) { best = keys[e]; who = e; }
            warp_best(best, who);
            if (best == -INFINITY) break;
            if ((uint32_t)lane == j) chosen = (int32_t)who;
            if (lane == 0) keys[who] = -INFINITY;
            __syncwarp();
        }
        double w = 0.0;
        const float l = chosen >= 0 ? load_logit<kType>(row, chosen) : -INFINITY;
        if (p.renormalise) {
            // Ratios of scores, formed from differences of their logarithms so that they survive scores too small to represent.
            const double log_score = chosen < 0 ? -INFINITY : p.sigmoid ? log_sigmoid(l) : (double)l;
            double most = log_score;
#pragma unroll
            for (int o = 16; o; o >>= 1) most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
            w = chosen < 0 ? 0.0 : exp(log_score - most);
            const double sum = warp_sum(w);
            w = chosen < 0 ? 0.0 : w / sum;
        } else if (chosen >= 0) {
            w = p.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : exp((double)l - top_logit) / total;
        }
        if ((uint32_t)lane < p.top) {
            weights[token * p.top + lane] = (float)(w * p.scale);
            ids[token * p.top + lane] = chosen;
        }
        __syncwarp();
    }
}

template <uint32_t kType>
__global__ void __launch_bounds__(kWarps * 32) route_gradient_kernel(const RouteDev p, const float *weights_grad, const int32_t *ids, float *logits_grad) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint64_t token = (uint64_t)blockIdx.x * kWarps + warp; token < p.tokens; token += (uint64_t)gridDim.x * kWarps) {
        const uint8_t *row = p.logits + token * p.stride;
        float *out = logits_grad + token * p.experts;
        int32_t id = (uint32_t)lane < p.top ? ids[token * p.top + lane] : -1;
        if (id >= (int32_t)p.experts) id = -1;
        const float l = id >= 0 ? load_logit<kType>(row, id) : -INFINITY;
        if (l == -INFINITY) id = -1;  // a masked expert has score 0 whatever its logit: no gradient
        const double g = id >= 0 ? (double)weights_grad[token * p.top + lane] * p.scale : 0.0;
        float top_logit = -INFINITY;
        double total = 0.0;
        if (!p.sigmoid && !p.renormalise) {
            for (uint32_t e = lane; e < p.experts; e += 32) top_logit = fmaxf(top_logit, load_logit<kType>(row, e));
            top_logit = warp_max(top_logit);
            for (uint32_t e = lane; e < p.experts; e += 32) {
                const float v = load_logit<kType>(row, e);
                if (v > -INFINITY) total += exp((double)v - top_logit);
            }
            total = warp_sum(total);
        }
        // d: the gradient that reaches this slot's logit through the slot itself; spread: what every logit gets in proportion to its score.
        double d = 0.0, spread = 0.0;
        if (p.renormalise) {
            const double log_score = id < 0 ? -INFINITY : p.sigmoid ? log_sigmoid(l) : (double)l;
            double most = log_score;
#pragma unroll
            for (int o = 16; o; o >>= 1) most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
            const double part = id < 0 ? 0.0 : exp(log_score - most), sum = warp_sum(part);
            const double u = id < 0 ? 0.0 : part / sum;
            const double mean = warp_sum(g * u);
            d = u * (g - mean);
            if (p.sigmoid) d *= id < 0 ? 0.0 : 1.0 / (1.0 + exp((double)l));  // 1 - s
        } else {
            const double s = id < 0 ? 0.0 : p.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : exp((double)l - top_logit) / total;
            d = p.sigmoid ? g * s * (id < 0 ? 0.0 : 1.0 / (1.0 + exp((double)l))) : g * s;
            if (!p.sigmoid) spread = warp_sum(d);
        }
        for (uint32_t e0 = 0; e0 < p.experts; e0 += 32) {
            const uint32_t e = e0 + lane;
            double v = 0.0;
            if (spread != 0.0 && e < p.experts) {
                const float x = load_logit<kType>(row, e);
                if (x > -INFINITY) v = -spread * exp((double)x - top_logit) / total;
            }
            for (uint32_t j = 0; j < p.top; ++j) {  // in order of the slots, so that an expert named twice gets the same sum every time
                const int32_t who = __shfl_sync(0xffffffffu, id, j);
                const double add = __shfl_sync(0xffffffffu, d, j);
                if (who == (int32_t)e) v += add;
            }
            if (e < p.experts) out[e] = (float)v;
        }
    }
}

uint32_t route_grid(uint64_t tokens) {
    const uint64_t blocks = (tokens + kWarps - 1) / kWarps;
    return (uint32_t)(blocks < 148ull * 64 ? blocks : 148ull * 64);
}

RouteDev route_dev(const RouteArgs &a) {
    return RouteDev{static_cast<const uint8_t *>(a.logits), a.logits_stride, a.tokens, a.experts, a.groups, a.top_groups, a.top, a.scale, a.bias, a.sigmoid, a.renormalise};
}

} // namespace

cudaError_t launch_route(const RouteArgs &a, float *weights, int32_t *ids, cudaStream_t stream) {
    const RouteDev p = route_dev(a);
    const uint32_t grid = route_grid(a.tokens), smem = kWarps * a.experts * sizeof(double);
    switch (a.type) {
    case kF32: route_kernel<kF32><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids); break;
    case kBF16: route_kernel<kBF16><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids); break;
    case kF16: route_kernel<kF16><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_route_gradient(const RouteArgs &a, const float *weights_grad, const int32_t *ids, float *logits_grad, cudaStream_t stream) {
    const RouteDev p = route_dev(a);
    const uint32_t grid = route_grid(a.tokens);
    switch (a.type) {
    case kF32: route_gradient_kernel<kF32><<<grid, kWarps * 32, 0, stream>>>(p, weights_grad, ids, logits_grad); break;
    case kBF16: route_gradient_kernel<kBF16><<<grid, kWarps * 32, 0, stream>>>(p, weights_grad, ids, logits_grad); break;
    case kF16: route_gradient_kernel<kF16><<<grid, kWarps * 32, 0, stream>>>(p, weights_grad, ids, logits_grad); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

} // namespace nkb
