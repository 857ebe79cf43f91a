// Routing of tokens to experts: scores from logits, selection, weights, and the gradient that trains the router.
//
//   score   s_e = softmax(l)_e or 1 / (1 + exp(-l_e))
//   choice  key_e = s_e + bias_e; with groups, a group is worth the sum of its two best keys and only the `top_groups` best
//           groups stay open; the `top` best open keys are chosen, best first, ties (of groups and of experts) to the lower index
//   weight  w_j = scale * s_{i_j}, or scale * s_{i_j} / sum over the chosen
//
// A logit of -infinity or NaN masks its expert: it has score 0 and is never chosen. A bias of -infinity or NaN only keeps its
// expert from being chosen. +infinity counts as the largest finite value. Slots that find no expert get id -1 and weight 0.
// Which of two near keys is the larger decides who is chosen, so keys are compared in 64 bits. Scores grow with their logits: without
// groups and with no bias, or one that is the same for all experts it does not bar, the logits themselves are compared, which keep
// their order where 64 bits no longer tell the scores apart (sigmoids of 40 and 50).
//
// Gradient, with p the chosen scores, g the incoming gradient times the scale and S their sum:
//   renormalised   d s_{i_j} = (g_j - sum_i g_i p_i / S) / S,   otherwise d s_{i_j} = g_j
//   softmax        d l_e = s_e (d s_e - sum_i d s_i s_i),       sigmoid d l_e = s_e (1 - s_e) d s_e
//
// Exponentials of scores that are given out are taken in 32 bits (off by three half steps at most, the rounding of their argument made good
// for) and summed in 64: a weight is within 8 half steps of f32 of its value, a gradient within 16 of the sum of its terms' magnitudes.
#include <cfloat>
#include "nkb_decode.cuh"
#include "nkb_mx.h"

namespace nkb {

namespace {

constexpr int kWarps = 4;

struct RouteDev {
    const uint8_t *logits;
    uint64_t stride;
    uint32_t tokens, experts, groups, top_groups, top;
    uint32_t width;                // lanes for one token's slots: 8, 16 or 32
    float scale;
    const float *bias;
    bool sigmoid, renormalise;
};

template <uint32_t kType>
__device__ __forceinline__ float load_logit(const uint8_t *row, uint32_t e) {
    float v;
    if constexpr (kType == kF32) v = reinterpret_cast<const float *>(row)[e];
    else v = decode_bits<kType>(reinterpret_cast<const uint16_t *>(row)[e]);
    return v == v ? fminf(v, FLT_MAX) + 0.0f : -INFINITY;  // NaN masks; -0 becomes 0
}
// -infinity bars the expert.
__device__ __forceinline__ float load_bias(const float *bias, uint32_t e) {
    const float b = bias ? __ldg(bias + e) : 0.0f;
    return b > -INFINITY ? fminf(b, FLT_MAX) : -INFINITY;  // false for NaN
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
// The largest key of the warp and its index; the lower index where keys are equal. (No key is -0.)
__device__ __forceinline__ void warp_best(double &key, uint32_t &index) {
    const long long bits = __double_as_longlong(key);
    const unsigned long long ordered = bits < 0 ? ~(unsigned long long)bits : (unsigned long long)bits | (1ull << 63);
    const uint32_t high = (uint32_t)(ordered >> 32), low = (uint32_t)ordered;
    const uint32_t best_high = __reduce_max_sync(0xffffffffu, high), best_low = __reduce_max_sync(0xffffffffu, high == best_high ? low : 0u);
    index = __reduce_min_sync(0xffffffffu, high == best_high && low == best_low ? index : 0xffffffffu);
    const unsigned long long best = ((unsigned long long)best_high << 32) | best_low;
    key = __longlong_as_double((long long)(best >> 63 ? best & ~(1ull << 63) : ~best));
}
__device__ __forceinline__ double sigmoid64(double l) { return 1.0 / (1.0 + exp(-l)); }
__device__ __forceinline__ double log_sigmoid(double l) { return fmin(l, 0.0) - log1p(exp(-fabs(l))); }

// A selected or doubtful expert's score in 64 bits, and the ratio of two sigmoids that vanish. The paths that need them are taken
// rarely, so that what they cost is the fetching of their instructions: one copy of each, outside the loops.
__device__ __noinline__ double exact_score(bool sigmoid, float l, float top_logit, double total) {
    const double e = exp(sigmoid ? -(double)l : (double)l - top_logit);
    return (sigmoid ? 1.0 : e) / (sigmoid ? 1.0 + e : total);
}
__device__ __noinline__ double small_sigmoid(float l, float largest) {
    return largest > -700.0f ? sigmoid64(l) : exp(log_sigmoid(l) - log_sigmoid(largest));
}

// exp(a - b) for a <= b in f32, the rounding of the difference made good for.
__device__ __forceinline__ float exp_difference(float a, float b) {
    const float d = a - b, t = d - a, lost = (a - (d - t)) - (b + t);
    return lost == lost ? fmaf(expf(d), lost, expf(d)) : expf(d);  // the correction is NaN where the difference overflows
}

// 1 / x for a positive x in the range of f32, to 46 bits: a 32-bit start and one step of Newton's.
__device__ __forceinline__ double reciprocal(double x) {
    const double r = (double)__frcp_rn((float)x);
    return r * fma(-x, r, 2.0);
}
// A chosen expert's score, up to the softmax's common factor, from one 32-bit exponential (off by two half units at most, the
// rest is 64 bits). Sigmoids of logits below -80 need the 64-bit exponential: see the callers.
__device__ __forceinline__ double fast_score(bool sigmoid, float l, float most) {
    return sigmoid ? reciprocal(1.0 + (double)expf(-l)) : (double)exp_difference(l, most);
}

// The logits lane * kPer .. of a token's row, -infinity where there is none or it is masked.
template <uint32_t kType, int kPer>
__device__ __forceinline__ void load_logits(const uint8_t *row, uint32_t experts, int lane, float (&l)[kPer]) {
    constexpr int kBytes = kType == kF32 ? 4 : 2, kLaneBytes = kPer * kBytes, kVector = kLaneBytes < 16 ? kLaneBytes : 16;
    const uint32_t first = lane * kPer;
    if (kVector >= 4 && first + kPer <= experts && (reinterpret_cast<uintptr_t>(row) & (kVector - 1)) == 0) {
        uint32_t w[(kLaneBytes + 3) / 4];
        const uint8_t *from = row + first * kBytes;
        if constexpr (kVector == 16) {
#pragma unroll
            for (int i = 0; i < kLaneBytes / 16; ++i) {
                const uint4 v = __ldg(reinterpret_cast<const uint4 *>(from) + i);
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        } else if constexpr (kVector == 8) {
            const uint2 v = __ldg(reinterpret_cast<const uint2 *>(from));
            w[0] = v.x; w[1] = v.y;
        } else if constexpr (kVector == 4) {
            w[0] = __ldg(reinterpret_cast<const uint32_t *>(from));
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            float v;
            if constexpr (kType == kF32) v = __uint_as_float(w[i]);
            else v = decode_bits<kType>(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
            l[i] = v == v ? fminf(v, FLT_MAX) + 0.0f : -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) l[i] = first + i < experts ? load_logit<kType>(row, first + i) : -INFINITY;
    }
}

// Batcher's odd-even merge network: `v` in descending order.
template <int kCount>
__device__ __forceinline__ void sort_descending(uint32_t (&v)[kCount]) {
#pragma unroll
    for (int p = 1; p < kCount; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j <= kCount - 1 - k; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i <= kCount - j - k - 1 && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t a = v[i + j], b = v[i + j + k];
                        v[i + j] = max(a, b);
                        v[i + j + k] = min(a, b);
                    }
}

// The choice in 64 bits, for the tokens whose keys 32 bits leave undecided. `keys`: room for one key per expert. Returns lane j's choice.
template <uint32_t kType>
__device__ __noinline__ int32_t choose_exactly(const RouteDev &p, const uint8_t *row, bool by_logit, double *keys, int lane) {
    double total = 0.0;
    float top_logit = -INFINITY;
    if (!p.sigmoid && !by_logit) {
        for (uint32_t e = lane; e < p.experts; e += 32) top_logit = fmaxf(top_logit, load_logit<kType>(row, e));
        top_logit = warp_max(top_logit);
        for (uint32_t e = lane; e < p.experts; e += 32) {
            const float l = load_logit<kType>(row, e);
            if (l > -INFINITY) total += exact_score(false, l, top_logit, 1.0);
        }
        total = warp_sum(total);
    }
    for (uint32_t e = lane; e < p.experts; e += 32) {
        const float l = load_logit<kType>(row, e), b = load_bias(p.bias, e);
        keys[e] = !(l > -INFINITY && b > -INFINITY) ? -INFINITY : by_logit ? (double)l : exact_score(p.sigmoid, l, top_logit, total) + b;
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
        for (uint32_t g = 0; g < p.top_groups; ++g) {
            double best = worth;
            uint32_t who = lane;
            warp_best(best, who);
            if (best == -INFINITY) break;
            if (who == (uint32_t)lane) { open = true; worth = -INFINITY; }
        }
        if ((uint32_t)lane < p.groups && !open)
            for (uint32_t i = 0; i < size; ++i) keys[lane * size + i] = -INFINITY;
        __syncwarp();
    }
    int32_t chosen = -1;
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
    return chosen;
}

// The `top` best of `count` candidates (one per lane) by their keys in 64 bits, in order, ties to the lower index. Returns lane j's choice.
template <uint32_t kType>
__device__ __noinline__ int32_t order_exactly(const RouteDev &p, const uint8_t *row, bool by_logit, int32_t chosen, uint32_t count, int32_t *places, int lane) {
    double total = 1.0;
    float top_logit = 0.0f;
    if (!by_logit && !p.sigmoid) {
        top_logit = -INFINITY;
        for (uint32_t e = lane; e < p.experts; e += 32) top_logit = fmaxf(top_logit, load_logit<kType>(row, e));
        top_logit = warp_max(top_logit);
        total = 0.0;
#pragma unroll 1
        for (uint32_t e = lane; e < p.experts; e += 32) total += exact_score(false, load_logit<kType>(row, e), top_logit, 1.0);
        total = warp_sum(total);
    }
    double key = -INFINITY;
    if (chosen >= 0) {
        const float l = load_logit<kType>(row, chosen);
        key = by_logit ? (double)l : exact_score(p.sigmoid, l, top_logit, total) + load_bias(p.bias, chosen);
    }
    uint32_t rank = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < count; ++i) {
        const double other = __shfl_sync(0xffffffffu, key, i);
        const int32_t who = __shfl_sync(0xffffffffu, chosen, i);
        rank += who >= 0 && (other > key || (other == key && who < chosen));
    }
    places[lane] = -1;
    __syncwarp();
    if (chosen >= 0) places[rank] = chosen;
    __syncwarp();
    return lane < (int)p.top ? places[lane] : -1;
}

// The choice where the last place is in question: everyone in an open group whose 32-bit key is not below `threshold` takes a lane, and
// those are put in order in 64 bits. -2 in all lanes where they are more than 32.
template <uint32_t kType, uint32_t kIndexBits>
__device__ __noinline__ int32_t choose_near(const RouteDev &p, const uint8_t *row, bool by_logit, uint32_t threshold, uint32_t open_groups, float least, float per_key, int32_t *places,
                                                int lane) {
    const bool direct = p.bias == nullptr && p.groups == 1;
    const uint32_t size = p.experts / p.groups;
    float top_logit = 0.0f, scaled = per_key;
    if (!direct && !p.sigmoid) {
        float total = 0.0f;
        top_logit = -INFINITY;
        for (uint32_t e = lane; e < p.experts; e += 32) top_logit = fmaxf(top_logit, load_logit<kType>(row, e));
        top_logit = warp_max(top_logit);
        for (uint32_t e = lane; e < p.experts; e += 32) total += expf(load_logit<kType>(row, e) - top_logit);
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        scaled = __fdividef(per_key, total);
    }
    uint32_t count = 0;
    int32_t candidate = -1;
    for (uint32_t base = 0; base < p.experts; base += 32) {
        const uint32_t e = base + lane;
        const float l = e < p.experts ? load_logit<kType>(row, e) : -INFINITY, b = e < p.experts ? load_bias(p.bias, e) : -INFINITY;
        bool in = l > -INFINITY && b > -INFINITY && ((open_groups >> (e / size)) & 1u);
        if (direct) in = in && (selection_key(l) >> kIndexBits) >= threshold;
        else {
            const float part = p.sigmoid ? __fdividef(1.0f, 1.0f + __expf(-l)) : expf(l - top_logit);
            in = in && __float2uint_rz(fmaf(part, scaled, (b - least) * per_key)) + 1u >= threshold;
        }
        const uint32_t found = __ballot_sync(0xffffffffu, in), many = __popc(found);
        if (count + many > 32) return -2;
        if ((uint32_t)lane >= count && (uint32_t)lane < count + many) candidate = (int32_t)(base + __fns(found, 0, lane - count + 1));
        count += many;
    }
    return order_exactly<kType>(p, row, by_logit, candidate, count, places, lane);
}

// One warp per token; lane i holds the experts i * kPer .. in registers.
//
// A key and its expert share one 32-bit word: the key in fixed point above, 31 - e of the warp's width below, so that one integer
// maximum over the warp finds the next choice and gives ties to the lower index. The fixed point comes from scores in 32 bits;
// `slack` bounds, in its units, how far it is off. Where every decision (chosen against next, open group against closed) is wider
// than that, or is a tie of equal inputs, the choice is the one 64 bits would make; otherwise those that may
// be chosen are put in order in 64 bits, or, where groups are in question, the whole choice is made there (choose_exactly). Keys that are the logits themselves (no bias, no groups) are the upper bits of their
// order-preserving integers, exact for 16-bit logits.
//
// 64 bits wait until a warp's batch is through: with the calls inside the loop its registers went to the stack around them. (At these
// register bounds up to 44 bytes a thread still do, for up to eight keys a lane.)
//
// 16,384 tokens x 256 experts, sigmoid, 4 of 8 groups, 8 chosen: 73 us with every token in 64 bits, 38 us with 32-bit keys whose expert was
// looked up in every round, 26 to 27 us now. 19 of these are about 700 instructions a token, a third of what the SMs can issue (the chain
// of one maximum after the other; more warps with fewer registers each were no faster); the rest is the last warps' way through 64 bits.
// Register bounds: 72 instead of 96 for eight keys a lane took 24 us to 20 without the 64-bit part, 64 was slower again.
template <uint32_t kType, int kPer>
__global__ void __launch_bounds__(kWarps * 32, kPer <= 4 ? 8 : kPer == 8 ? 7 : kPer == 16 ? 4 : 2) route_kernel(const RouteDev p, float *weights, int32_t *ids) {
    constexpr uint32_t kIndexBits = kPer == 1 ? 5 : kPer == 2 ? 6 : kPer == 4 ? 7 : kPer == 8 ? 8 : kPer == 16 ? 9 : 10;
    constexpr bool kSorted = kPer <= 8;  // each lane keeps its keys in order; beyond that the network costs more than it saves
    constexpr uint32_t kWidth = 32 * kPer, kUnits = (1u << (32 - kIndexBits)) - 64;  // some room above for rounding
    extern __shared__ double keys_all[];
    __shared__ int32_t places_all[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto expert_of = [](uint32_t word) { return kWidth - 1 - (word & (kWidth - 1)); };
    const bool direct = p.bias == nullptr && p.groups == 1;
    const uint32_t size = p.experts / p.groups, lanes = size / kPer;
    const bool whole_lanes = size % kPer == 0 && (lanes & (lanes - 1)) == 0;  // a group is a power of two of lanes
    // Scores lie in [0, 1], keys in [least bias, 1 + most bias]. zero_key: the units of a key of 0.
    float bias[kPer], least = INFINITY, most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const uint32_t e = lane * kPer + i;
        bias[i] = e < p.experts ? load_bias(p.bias, e) : -INFINITY;
        if (bias[i] > -INFINITY) { least = fminf(least, bias[i]); most = fmaxf(most, bias[i]); }
    }
    least = -warp_max(-least);
    most = warp_max(most);
    const bool by_logit = p.groups == 1 && (p.bias == nullptr || __all_sync(0xffffffffu, !(least < most)));
    if (!(least <= most)) least = most = 0.0f;  // every expert is barred
    least = fminf(least, 0.0f);                 // so that a key of 0 is on the scale
    const bool workable = direct || (fabsf(least) < 16.0f && fabsf(most) < 16.0f);  // wider biases leave the scale too coarse
    const float per_key = (float)kUnits / (1.0f + (most - least)), zero_key = -least * per_key;
    // A score is off by a few units of its last place (exp, division), the softmax's sum one more per addition (and its scores are at most
    // 1 / sum); the sum with the bias and the step to fixed point round four times more.
    const float score_error = (p.sigmoid ? 8.0f : (float)(kPer + 16)) * 0x1p-23f * per_key, bias_error = (fabsf(least) + fabsf(most)) * 0x1p-23f * per_key + 8.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) bias[i] = (bias[i] - least) * per_key;  // -infinity stays
    // A warp chooses for `batch` tokens one after the other and then works out their weights together, `width` lanes each.
    const uint32_t width = p.width, batch = 32 / width, place = lane / width, slot = lane % width;
    const uint32_t step = gridDim.x * kWarps * batch;
    for (uint32_t first = (blockIdx.x * kWarps + warp) * batch; first < p.tokens; first += step) {
    int32_t chosen_all = -1;         // lane place * width + j: slot j of token first + place
    float top_all = 0.0f;            // that token's largest logit, and the sum of its exponentials: the softmax without renormalisation
    double total_all = 1.0;
    float logit[kPer], next[kPer];
    load_logits<kType, kPer>(p.logits + first * p.stride, p.experts, lane, logit);
    uint32_t unsure = 0;             // tokens of the batch that want 64 bits, and lane t: for the whole choice (0), the order of the chosen
    uint32_t how = 0, among = 0;     // (all ones), or the choice from a threshold on, among these groups
    for (uint32_t t = 0; t < batch && first + t < p.tokens; ++t) {
        const uint8_t *row = p.logits + (first + t) * p.stride;
        if (t + 1 < batch && first + t + 1 < p.tokens) load_logits<kType, kPer>(row + p.stride, p.experts, lane, next);
        float top_logit = -INFINITY;
        if (!p.sigmoid) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) top_logit = fmaxf(top_logit, logit[i]);
            top_logit = warp_max(top_logit);
        }
        uint32_t key[kPer], slack = 0, open_groups = 1;
        const uint32_t last = kWidth - 1 - lane * kPer;
        if (direct) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) key[i] = logit[i] > -INFINITY ? (selection_key(logit[i]) & ~(kWidth - 1)) | (last - i) : 0u;
        } else {
            float scaled = per_key, largest_score = 1.0f;
            float part[kPer];
            if (p.sigmoid) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) part[i] = __fdividef(1.0f, 1.0f + __expf(-logit[i]));
            } else {
                float total = 0.0f;
#pragma unroll
                for (int i = 0; i < kPer; ++i) { part[i] = expf(logit[i] - top_logit); if (logit[i] > -INFINITY) total += part[i]; }
#pragma unroll
                for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
                scaled = __fdividef(per_key, total);
                largest_score = __fdividef(1.0f, total);
            }
            slack = (uint32_t)fmaf(score_error, largest_score, bias_error) + 1u;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const float units = fmaf(part[i], scaled, bias[i]);
                // One unit up: 0 stands for no key.
                key[i] = logit[i] > -INFINITY && units > -INFINITY ? ((__float2uint_rz(units) + 1u) << kIndexBits) | (last - i) : 0u;
            }
        }
        if constexpr (kSorted) sort_descending(key);
        bool sure = workable;
        if (p.groups > 1) {
            uint32_t worth = 0;  // lane g: group g's, in units; 0 where nobody is left
            const uint32_t alone = (uint32_t)zero_key;  // keeps sums of one and of two keys comparable
            auto worth_of = [&](uint32_t first, uint32_t second) {
                if (first == 0) return 0u;
                const uint32_t a = first >> kIndexBits, b = second ? second >> kIndexBits : alone;
                return (a >> 1) + (b >> 1) + 1u;  // half units: the sum fits 32 bits
            };
            if (whole_lanes) {
                uint32_t first = key[0], second = 0;
#pragma unroll
                for (int i = 1; i < (kSorted && kPer > 2 ? 2 : kPer); ++i) {
                    second = max(second, min(first, key[i]));
                    first = max(first, key[i]);
                }
                for (uint32_t o = 1; o < lanes; o <<= 1) {
                    const uint32_t f = __shfl_xor_sync(0xffffffffu, first, o), n = __shfl_xor_sync(0xffffffffu, second, o);
                    second = max(min(first, f), max(second, n));
                    first = max(first, f);
                }
                worth = __shfl_sync(0xffffffffu, worth_of(first, second), lane * lanes);
            } else {
                for (uint32_t g = 0; g < p.groups; ++g) {
                    uint32_t first = 0, second = 0;
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const uint32_t e = expert_of(key[i]), k = e >= g * size && e < (g + 1) * size ? key[i] : 0u;
                        second = max(second, min(first, k));
                        first = max(first, k);
                    }
                    const uint32_t best = __reduce_max_sync(0xffffffffu, first);  // keys differ from one another in their experts
                    const uint32_t behind = __reduce_max_sync(0xffffffffu, first == best ? second : first);
                    if (lane == (int)g) worth = worth_of(best, behind);
                }
            }
            if ((uint32_t)lane >= p.groups) worth = 0;
            uint32_t rank = 0;
            for (uint32_t g = 0; g < p.groups; ++g) {
                const uint32_t other = __shfl_sync(0xffffffffu, worth, g);
                rank += other > worth || (other == worth && (int)g < lane);
            }
            const bool open = (uint32_t)lane < p.groups && rank < p.top_groups;
            const uint32_t least_open = __reduce_min_sync(0xffffffffu, open ? worth : 0xffffffffu);
            const uint32_t most_closed = __reduce_max_sync(0xffffffffu, open ? 0u : worth);
            // A worth is off by two keys' errors, halved, and its roundings.
            if (most_closed != 0 && least_open - most_closed <= 2 * slack + 4) sure = false;
            open_groups = __ballot_sync(0xffffffffu, open);
            if (whole_lanes) {
                if (!((open_groups >> (lane / lanes)) & 1u)) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) key[i] = 0u;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (key[i] != 0u && !((open_groups >> (expert_of(key[i]) / size)) & 1u)) key[i] = 0u;
                if constexpr (kSorted) sort_descending(key);
            }
        }
        // Lane j takes the j-th word; one more is looked at, since it has to be further off than the error, too.
        const uint32_t unsure_at = direct ? 0u : 2 * slack;
        uint32_t word = 0, behind = 0;
        for (uint32_t j = 0; j <= p.top; ++j) {
            uint32_t mine = key[0];
            if constexpr (!kSorted) {
#pragma unroll
                for (int i = 1; i < kPer; ++i) mine = max(mine, key[i]);
            }
            behind = __reduce_max_sync(0xffffffffu, mine);
            if (behind == 0) break;
            if (mine == behind) {
                if constexpr (kSorted) {
#pragma unroll
                    for (int i = 0; i + 1 < kPer; ++i) key[i] = key[i + 1];
                    key[kPer - 1] = 0u;
                } else {
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        if (key[i] == behind) key[i] = 0u;
                }
            }
            if (lane == (int)j) word = behind;
        }
        auto undecided = [&](uint32_t ahead, uint32_t then) {  // closer than the error, and not a tie of equal inputs
            if (then == 0 || (ahead >> kIndexBits) - (then >> kIndexBits) > unsure_at) return false;
            const uint32_t x = expert_of(ahead), y = expert_of(then);
            return !(load_logit<kType>(row, x) == load_logit<kType>(row, y) && load_bias(p.bias, x) == load_bias(p.bias, y));
        };
        const uint32_t before = __shfl_up_sync(0xffffffffu, word, 1);
        bool ordered = !__any_sync(0xffffffffu, lane > 0 && undecided(before, word));
        // A tie of the last one chosen may hide others behind it that are near and not a tie. (Keys that are 16-bit logits are exact.)
        if (kType == kF32 || !direct) {
            const bool edge = p.top == 32 ? behind != 0 : lane == (int)p.top && word != 0 && (before >> kIndexBits) - (word >> kIndexBits) <= unsure_at;
            if (__any_sync(0xffffffffu, edge) && ordered) {
                const uint32_t last_word = __shfl_sync(0xffffffffu, word, p.top - 1);
                bool near = p.top == 32 && undecided(last_word, behind);
#pragma unroll
                for (int i = 0; i < kPer; ++i) near = near || undecided(last_word, key[i]);
                ordered = !__any_sync(0xffffffffu, near);
            }
        }
        int32_t chosen = word != 0 && lane < (int)p.top ? (int32_t)expert_of(word) : -1;
        if (!sure || !ordered) {
            const uint32_t last = __shfl_sync(0xffffffffu, word, p.top - 1) >> kIndexBits;
            const bool last_clear = behind == 0 || last - (behind >> kIndexBits) > unsure_at;
            unsure |= 1u << t;
            if (lane == (int)t) {
                how = !sure ? 0u : last_clear ? 0xffffffffu : last > unsure_at + 2 ? last - unsure_at - 2 : 1u;
                among = open_groups;
            }
        }
        const int32_t mine_of = __shfl_sync(0xffffffffu, chosen, slot);
        if (place == t) chosen_all = mine_of;
        if (!p.sigmoid && !p.renormalise) {
            double total = 0.0;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (logit[i] > -INFINITY) total += (double)exp_difference(logit[i], top_logit);
            total = warp_sum(total);
            if (place == t) { top_all = top_logit; total_all = total; }
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) logit[i] = next[i];
    }
    for (; unsure; unsure &= unsure - 1) {
        const uint32_t t = __ffs(unsure) - 1, what = __shfl_sync(0xffffffffu, how, t), groups = __shfl_sync(0xffffffffu, among, t);
        const uint8_t *row = p.logits + (first + t) * p.stride;
        int32_t chosen = -2;
        if (what == 0xffffffffu) {
            chosen = __shfl_sync(0xffffffffu, chosen_all, t * width + (lane & (width - 1)));
            chosen = order_exactly<kType>(p, row, by_logit, lane < (int)p.top ? chosen : -1, p.top, places_all[warp], lane);
        } else if (what != 0) {
            chosen = choose_near<kType, kIndexBits>(p, row, by_logit, what, groups, least, per_key, places_all[warp], lane);
        }
        if (__any_sync(0xffffffffu, chosen == -2)) {
            chosen = choose_exactly<kType>(p, row, by_logit, keys_all + (size_t)warp * p.experts, lane);
            __syncwarp();
        }
        const int32_t mine_of = __shfl_sync(0xffffffffu, chosen, slot);
        if (place == t) chosen_all = mine_of;
    }
    const uint64_t token = first + place;
    const float l = chosen_all >= 0 ? load_logit<kType>(p.logits + token * p.stride, chosen_all) : -INFINITY;
    const uint32_t small = p.sigmoid ? __ballot_sync(0xffffffffu, chosen_all >= 0 && l < -80.0f) : 0u;
    const bool near_zero = ((small >> (place * width)) & (0xffffffffu >> (32 - width))) != 0;  // in this token
    double w = 0.0;
    if (p.renormalise) {
        // Scores as they are while they can be represented, ratios from differences of logarithms where they vanish.
        float largest = l;
        if (!p.sigmoid || small != 0)
            for (uint32_t o = 1; o < width; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        if (chosen_all >= 0) w = !near_zero ? fast_score(p.sigmoid, l, largest) : small_sigmoid(l, largest);
        double sum = w;
        for (uint32_t o = 1; o < width; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (chosen_all >= 0) w *= sum > 1e-30 ? reciprocal(sum) : 1.0 / sum;
    } else if (p.sigmoid) {
        if (chosen_all >= 0) w = near_zero ? small_sigmoid(l, 0.0f) : fast_score(true, l, 0.0f);
    } else if (chosen_all >= 0) {
        w = (double)exp_difference(l, top_all) * reciprocal(total_all);
    }
    if (slot < p.top && token < p.tokens) {
        weights[token * p.top + slot] = (float)(w * p.scale);
        ids[token * p.top + slot] = chosen_all;
    }
    }
}

// One warp per batch of one, two or four tokens, `width` lanes for the slots of each. What reaches a chosen expert's logit is worked out in
// 64 bits from the 32-bit exponentials, one slot per lane, and put into a row in shared memory; the rows then go out in whole lines. Only
// the softmax without renormalisation gives every logit something.
//
// With n the scores' numerators (exponentials, or sigmoids), N their sum over the chosen, or over all experts without renormalisation, and
// O the part of it that was not chosen, the gradient of a chosen logit is
//   n_e / N^2 (sum over the chosen j of n_j (g_e - g_j) + g_e O), for sigmoids times 1 - s_e.
// Where one score is nearly all of N the terms of g_e N - sum of n_j g_j cancel. So every g is taken relative to that of the largest
// numerator first (relative to 0 if that is not among the chosen), which leaves the bracket as it is and takes its largest terms out.
// Bound by the write of the rows and the start: 16,384 x 256 f32, sigmoid, 8 chosen, 5.8 us for 18 MB (2.7 us at the copy rate); 16,384 x 64
// bf16, softmax renormalised, 6 chosen, 4.1 us; 16 tokens 3.2 us. Softmax without renormalisation, which reads every logit: 16,384 x 256
// 14.0 us, 16,384 x 64 8.8 us (8.1 us with the subtraction of two 32-bit values, which lost what nearly cancels: a fifth of a chosen logit's
// gradient where it lies 18 above the others, all of it from 22 on).
template <uint32_t kType>
__global__ void __launch_bounds__(kWarps * 32) route_gradient_kernel(const RouteDev p, const float *weights_grad, const int32_t *ids, float *logits_grad) {
    extern __shared__ float rows_all[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t padded = (p.experts + 3) / 4 * 4;
    const uint32_t width = p.width, batch = 32 / width, place = lane / width, slot = lane % width;
    float *lines = rows_all + (size_t)warp * batch * padded, *line = lines + place * padded;
    const bool dense = !p.sigmoid && !p.renormalise;
    auto over_slots = [&](double v) {
        for (uint32_t o = 1; o < width; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    for (uint32_t first = (blockIdx.x * kWarps + warp) * batch; first < p.tokens; first += gridDim.x * kWarps * batch) {
        const uint64_t token = first + place;
        const uint32_t here = min(batch, p.tokens - first);
        int32_t id = -1;
        float l = -INFINITY, incoming = 0.0f;
        if (slot < p.top && token < p.tokens) {
            id = ids[token * p.top + slot];
            incoming = weights_grad[token * p.top + slot];
            if (id >= 0 && id < (int32_t)p.experts) l = load_logit<kType>(p.logits + token * p.stride, id);
        }
        if (!(l > -INFINITY)) id = -1;  // a masked expert has score 0 whatever its logit: no gradient
        const double g = id >= 0 ? (double)incoming * p.scale : 0.0;
        float top_logit = -INFINITY;
        double all = 0.0;  // the numerators of all experts
        if (dense) {
            for (uint32_t t = 0; t < here; ++t) {
                const uint8_t *row = p.logits + (first + t) * p.stride;
                float largest = -INFINITY;
                double sum = 0.0;
                for (uint32_t e = lane; e < p.experts; e += 32) largest = fmaxf(largest, load_logit<kType>(row, e));
                largest = warp_max(largest);
                for (uint32_t e = lane; e < p.experts; e += 32) {
                    const float v = load_logit<kType>(row, e), part = v > -INFINITY ? exp_difference(v, largest) : 0.0f;
                    lines[t * padded + e] = part;
                    sum += (double)part;
                }
                sum = warp_sum(sum);
                if (place == t) { top_logit = largest; all = sum; }
            }
            __syncwarp();
        } else {
            for (uint32_t i = lane; i < here * padded / 4; i += 32) reinterpret_cast<float4 *>(lines)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        // An expert named twice counts once in the softmax, with its slots' sum, in their order, in the first of them.
        const uint32_t segment = (width == 32 ? 0xffffffffu : (1u << width) - 1u) << (place * width);
        const uint32_t same = __match_any_sync(0xffffffffu, id) & segment;
        const bool first_of = id >= 0 && __ffs(same) - 1 == lane, twice = __any_sync(0xffffffffu, id >= 0 && __popc(same) > 1);
        auto over_same = [&](double v) {
            double sum = 0.0;
            for (uint32_t j = 0; j < width; ++j) {
                const double other = __shfl_sync(0xffffffffu, v, place * width + j);
                if ((same >> (place * width + j)) & 1u) sum += other;
            }
            return sum;
        };
        double d = 0.0;  // what this slot's logit gets through the slot itself
        const bool near_limit = p.sigmoid && ((__ballot_sync(0xffffffffu, id >= 0 && fabsf(l) > 80.0f) >> (place * width)) & (0xffffffffu >> (32 - width))) != 0;
        if (p.renormalise || dense) {
            double mine = dense && twice ? over_same(g) : g, part = 0.0;
            const bool counts = dense ? first_of : id >= 0;
            if (!counts) mine = 0.0;
            // The gradient that comes in at the slot with the largest logit; of several such the largest, so that no order matters.
            float most = counts ? l : -INFINITY;
            double ref = mine;
            for (uint32_t o = 1; o < width; o <<= 1) {
                const float other = __shfl_xor_sync(0xffffffffu, most, o);
                const double other_ref = __shfl_xor_sync(0xffffffffu, ref, o);
                if (other > most || (other == most && other_ref > ref)) { most = other; ref = other_ref; }
            }
            if (counts) part = dense ? (double)exp_difference(l, top_logit) : !near_limit ? fast_score(p.sigmoid, l, most) : small_sigmoid(l, most);
            const double chosen = over_slots(part);
            double others = 0.0;
            if (dense) {
                // The difference loses 20 of its 53 bits at most, or the others are added up by themselves.
                others = all - chosen;
                uint32_t rare = __ballot_sync(0xffffffffu, slot == 0 && others < all * 0x1p-20);
                if (rare != 0) {
                    if (counts) line[id] = 0.0f;
                    __syncwarp();
                    for (; rare; rare &= rare - 1) {
                        const uint32_t t = (__ffs(rare) - 1) / width;
                        double sum = 0.0;
                        for (uint32_t e = lane; e < p.experts; e += 32) sum += (double)lines[t * padded + e];
                        sum = warp_sum(sum);
                        if (place == t) others = sum;
                    }
                }
                if (most < top_logit || others > 1.0) ref = 0.0;  // the slot's numerator is 1 at most
            }
            if (!(fabs(ref) < INFINITY)) ref = 0.0;
            const double total = chosen + others, shifted = over_slots(part * (mine - ref)) - others * ref;
            const double inverse = total > 0.0 ? total > 1e-30 ? reciprocal(total) : 1.0 / total : 0.0;
            if (counts) d = part * inverse * (((mine - ref) * total - shifted) * inverse);
            if (dense) {
                const float per_part = (float)(-(over_slots(part * mine) * inverse) * inverse);
                for (uint32_t t = 0; t < here; ++t) {
                    const float factor = __shfl_sync(0xffffffffu, per_part, t * width);
                    for (uint32_t e = lane; e < p.experts; e += 32) lines[t * padded + e] *= factor;
                }
            }
        } else if (id >= 0) {
            d = g * (near_limit ? small_sigmoid(l, 0.0f) : fast_score(true, l, 0.0f));
        }
        if (p.sigmoid && id >= 0) d *= near_limit ? small_sigmoid(-l, 0.0f) : fast_score(true, -l, 0.0f);  // 1 - s
        if (!dense && twice) d = over_same(d);
        __syncwarp();
        if (first_of) line[id] = (float)d;
        __syncwarp();
        float *out = logits_grad + (uint64_t)first * p.experts;
        if ((p.experts & 3u) == 0 && (reinterpret_cast<uintptr_t>(logits_grad) & 15u) == 0)  // the rows lie one behind the other here and there
            for (uint32_t i = lane; i < here * (p.experts / 4); i += 32) __stcs(reinterpret_cast<float4 *>(out) + i, reinterpret_cast<const float4 *>(lines)[i]);
        else
            for (uint32_t t = 0; t < here; ++t)
                for (uint32_t e = lane; e < p.experts; e += 32) out[(uint64_t)t * p.experts + e] = lines[t * padded + e];
        __syncwarp();
    }
}

uint32_t route_grid(const RouteDev &p) {
    const uint64_t tokens = (uint64_t)kWarps * (32 / p.width), blocks = (p.tokens + tokens - 1) / tokens;
    return (uint32_t)(blocks < 148ull * 16 ? blocks : 148ull * 16);
}

RouteDev route_dev(const RouteArgs &a) {
    // Several tokens share a warp's 64-bit work where there are enough of them to fill the GPU all the same, and their rows of the
    // gradient 48 KiB.
    uint32_t width = a.tokens < 4096 || a.top > 16 ? 32 : a.top <= 8 ? 8 : 16;
    if (width == 8 && a.experts > 768) width = 16;
    return RouteDev{static_cast<const uint8_t *>(a.logits), a.logits_stride, (uint32_t)a.tokens, a.experts, a.groups, a.top_groups, a.top, width, a.scale, a.bias,
                    a.sigmoid, a.renormalise};
}

template <uint32_t kType>
void route_by_width(const RouteDev &p, float *weights, int32_t *ids, cudaStream_t stream) {
    const uint32_t grid = route_grid(p), smem = kWarps * p.experts * sizeof(double);
    if (p.experts <= 32) route_kernel<kType, 1><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids);
    else if (p.experts <= 64) route_kernel<kType, 2><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids);
    else if (p.experts <= 128) route_kernel<kType, 4><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids);
    else if (p.experts <= 256) route_kernel<kType, 8><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids);
    else if (p.experts <= 512) route_kernel<kType, 16><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids);
    else route_kernel<kType, 32><<<grid, kWarps * 32, smem, stream>>>(p, weights, ids);
}

} // namespace

cudaError_t launch_route(const RouteArgs &a, float *weights, int32_t *ids, cudaStream_t stream) {
    const RouteDev p = route_dev(a);
    switch (a.type) {
    case kF32: route_by_width<kF32>(p, weights, ids, stream); break;
    case kBF16: route_by_width<kBF16>(p, weights, ids, stream); break;
    case kF16: route_by_width<kF16>(p, weights, ids, stream); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_route_gradient(const RouteArgs &a, const float *weights_grad, const int32_t *ids, float *logits_grad, cudaStream_t stream) {
    const RouteDev p = route_dev(a);
    const uint32_t grid = route_grid(p), smem = kWarps * (32 / p.width) * ((a.experts + 3) / 4 * 4) * sizeof(float);
    switch (a.type) {
    case kF32: route_gradient_kernel<kF32><<<grid, kWarps * 32, smem, stream>>>(p, weights_grad, ids, logits_grad); break;
    case kBF16: route_gradient_kernel<kBF16><<<grid, kWarps * 32, smem, stream>>>(p, weights_grad, ids, logits_grad); break;
    case kF16: route_gradient_kernel<kF16><<<grid, kWarps * 32, smem, stream>>>(p, weights_grad, ids, logits_grad); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

} // namespace nkb
