// Routing of tokens to experts:
//
//   s   = sigmoid(l) or softmax(l) over all experts
//   key = s + bias, or the logit l itself when there is no bias (s rises with l)
//   with groups: the value of a group of consecutive experts is the sum of its two largest
//         keys (of s + bias; s without a bias) or its largest; experts outside the
//         `topk_groups` best groups are not eligible
//   idx = the k largest eligible keys, descending, ties to the lower expert
//   w   = s[idx], divided by their sum if asked for, times `scale`
//
// An expert whose logit is -inf or NaN, or whose bias is, is never chosen; a slot for which
// no expert is left gets index -1 (no route) and weight 0.  A logit of +inf counts as the
// largest finite float.
//
// The order is that of the keys computed in 64 bits, whatever the sums' order in 32: keys
// are kept as f32 with a bound on their error, and a round in which two candidates lie
// within that bound of each other computes those candidates again in f64.
//
// One warp per token; each of a group's lanes holds consecutive experts in registers, as
// integers that order like the floats (0 = not eligible), so that a round of the selection
// is one redux.max, a ballot, and a rescan of the winner's registers.  Bound by
// instruction issue for many tokens and by latency for few; the bytes (E logits in, 12 k
// out) are small beside both.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cfloat>
#include <stdint.h>

#include "device_common.cuh"
#include "ptx.cuh"

namespace gcmoe {

constexpr uint32_t kRouteWarps = 4;
constexpr uint32_t kRouteMaxPerLane = 64;
enum LogitType : uint32_t { kLogitF32 = 0, kLogitBf16 = 1, kLogitF16 = 2 };

struct RouteParams {
    const void* logits;
    const float* bias;            // f32 [E] or null
    long long* topk_idx;          // int64 [T][k]
    float* topk_weights;          // f32 [T][k]
    uint64_t logits_stride;       // elements between rows
    uint32_t num_tokens, num_experts, topk;
    uint32_t num_groups, topk_groups, group_size;
    uint32_t lanes_per_group;     // power of two; lanes_per_group * num_groups <= 32
    uint32_t per_lane;            // experts of a lane: ceil(group_size / lanes_per_group)
    uint32_t logit_type, sigmoid, group_by_max, renormalize;
    float scale;
};

// Integers in the order of the floats; -0 and +0 are the same, and no float maps to 0.
__device__ __forceinline__ uint32_t order_f32(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (b & 0x80000000u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unorder_f32(uint32_t u) {
    return __uint_as_float(u ^ (u & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t order_f64(double v) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return b ^ (b >> 63 ? 0xffffffffffffffffull : 0x8000000000000000ull);
}

// A row's logit, and whether the expert can be chosen at all.
__device__ __forceinline__ bool load_logit(const RouteParams& p, uint64_t row, uint32_t e, float& l, float& b) {
    if (p.logit_type == kLogitF32) l = static_cast<const float*>(p.logits)[row + e];
    else if (p.logit_type == kLogitBf16) l = __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[row + e]);
    else l = __half2float(static_cast<const __half*>(p.logits)[row + e]);
    l = fminf(l, isnan(l) ? l : FLT_MAX);
    b = p.bias != nullptr ? p.bias[e] : 0.f;
    return l > -INFINITY && b > -INFINITY;            // false for NaN too
}

__device__ __forceinline__ float sigmoid_f32(float l) {
    const float z = expf(-fabsf(l));
    return (l >= 0.f ? 1.f : z) / (1.f + z);
}

// Softmax statistics of the row: exact maximum, sum in 32 and (on demand) 64 bits.
struct RowStats {
    float top, sum;
    double sum64;
    bool has64;
};

template <int kPerLane>
__device__ __noinline__ double row_sum_f64(const RouteParams& p, uint64_t row, uint32_t first, uint32_t n, float top) {
    double sum = 0.0;
    for (uint32_t i = 0; i < n; ++i) {
        float l, b;
        if (load_logit(p, row, first + i, l, b)) sum += exp(double(l) - double(top));
    }
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
}

// The score plus bias in 64 bits.
__device__ __forceinline__ double key_f64(const RouteParams& p, const RowStats& s, float l, float b) {
    if (p.sigmoid) return 1.0 / (1.0 + exp(-double(l))) + double(b);
    return exp(double(l) - double(s.top)) / s.sum64 + double(b);
}

template <int kPerLane>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
    constexpr uint32_t kAll = 0xffffffffu;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t t = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    ptx::launch_dependents();
    ptx::grid_dependency_wait();
    if (t >= p.num_tokens) return;                    // whole warps

    const uint64_t row = t * p.logits_stride;
    const uint32_t group = lane / p.lanes_per_group, sub = lane % p.lanes_per_group;
    const uint32_t begin = sub * p.per_lane;
    const uint32_t n = group < p.num_groups && begin < p.group_size ? min(p.per_lane, p.group_size - begin) : 0u;
    const uint32_t first = group * p.group_size + begin;
    const bool has_bias = p.bias != nullptr;

    float value[kPerLane];                            // logits, then keys; -inf: not eligible
    float bias[kPerLane];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        value[i] = -INFINITY;
        bias[i] = 0.f;
        if (uint32_t(i) < n) {
            float l, b;
            if (load_logit(p, row, first + i, l, b)) { value[i] = l; bias[i] = b; }
        }
        top = fmaxf(top, value[i]);
    }

    const bool by_sum = p.num_groups > 1 && !p.group_by_max;
    RowStats stats = {0.f, 1.f, 1.0, false};
    if (!p.sigmoid && (has_bias || by_sum || !p.renormalize)) {
        // masked experts have no part in the softmax; an empty row keeps top = 0
#pragma unroll
        for (uint32_t d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, d));
        if (top > -INFINITY) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) sum += expf(value[i] - top);
#pragma unroll
            for (uint32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
            stats.top = top;
            stats.sum = sum;
        }
    }
    // Bound on the f32 error of a score: sigmoid, a few roundings of a value below one;
    // softmax, the sum's roundings (2048 terms at most, pairwise over lanes) and the exponent's.
    const float score_error = p.sigmoid ? 0x1p-21f : 0x1p-17f;
    const float inv_sum = 1.f / stats.sum;
    const bool keyed = has_bias;                      // keys are scores, not logits
    auto score = [&](float l) { return p.sigmoid ? sigmoid_f32(l) : expf(l - stats.top) * inv_sum; };
    auto need_sum64 = [&]() {
        if (!p.sigmoid && !stats.has64) {
            stats.sum64 = row_sum_f64<kPerLane>(p, row, first, n, stats.top);
            stats.has64 = true;
        }
    };

    bool eligible = true;                             // this lane's group is among the best
    if (p.num_groups > 1) {
        float a1 = -INFINITY, a2 = -INFINITY;         // the two largest members of the lane, then of the group
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const bool alive = value[i] > -INFINITY;
            const float m = !alive ? -INFINITY : (keyed || by_sum) ? score(value[i]) + bias[i] : value[i];
            if (keyed) value[i] = m;
            a2 = fmaxf(a2, fminf(a1, m));
            a1 = fmaxf(a1, m);
        }
        for (uint32_t d = p.lanes_per_group >> 1; d > 0; d >>= 1) {
            const float o1 = __shfl_xor_sync(kAll, a1, d), o2 = __shfl_xor_sync(kAll, a2, d);
            a2 = fmaxf(fminf(a1, o1), fmaxf(a2, o2));
            a1 = fmaxf(a1, o1);
        }
        const bool two = by_sum && a2 > -INFINITY;
        const float mine = two ? a1 + a2 : a1;
        // a group without eligible experts has value -inf; bounds of the others' errors
        float error = 0.f;
        if ((keyed || by_sum) && mine > -INFINITY && mine < INFINITY)
            error = (two ? 2.f : 1.f) * score_error + 0x1p-22f * (fabsf(a1) + (two ? fabsf(a2) : 0.f));
        uint32_t rank = 0;
        bool close = false;
        for (uint32_t o = 0; o < p.num_groups; ++o) {
            const float v = __shfl_sync(kAll, mine, o * p.lanes_per_group);
            const float e = __shfl_sync(kAll, error, o * p.lanes_per_group);
            rank += v > mine || (v == mine && o < group);
            close |= o != group && fabsf(v - mine) <= e + error;
        }
        if ((keyed || by_sum) && __any_sync(kAll, close && group < p.num_groups)) {
            need_sum64();
            double b1 = -INFINITY, b2 = -INFINITY;
            for (uint32_t i = 0; i < n; ++i) {
                float l, b;
                if (!load_logit(p, row, first + i, l, b)) continue;
                const double m = key_f64(p, stats, l, b);
                b2 = fmax(b2, fmin(b1, m));
                b1 = fmax(b1, m);
            }
            for (uint32_t d = p.lanes_per_group >> 1; d > 0; d >>= 1) {
                const double o1 = __shfl_xor_sync(kAll, b1, d), o2 = __shfl_xor_sync(kAll, b2, d);
                b2 = fmax(fmin(b1, o1), fmax(b2, o2));
                b1 = fmax(b1, o1);
            }
            const double exact = by_sum && b2 > -INFINITY ? b1 + b2 : b1;
            rank = 0;
            for (uint32_t o = 0; o < p.num_groups; ++o) {
                const double v = __shfl_sync(kAll, exact, o * p.lanes_per_group);
                rank += v > exact || (v == exact && o < group);
            }
        }
        eligible = rank < p.topk_groups;
    } else if (keyed) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (value[i] > -INFINITY) value[i] = score(value[i]) + bias[i];
    }

    uint32_t key[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) key[i] = eligible && value[i] > -INFINITY ? order_f32(value[i]) : 0u;

    uint32_t best = 0, second = 0, best_i = 0;        // this lane's two largest keys
    auto rescan = [&]() {
        best = second = best_i = 0;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const bool up = key[i] > best;            // equal keys: the first stays
            second = max(second, up ? best : key[i]);
            best_i = up ? i : best_i;
            best = up ? key[i] : best;
        }
    };
    rescan();
    int chosen = -1;                                  // lane j: the j-th choice
    for (uint32_t j = 0; j < p.topk; ++j) {
        const uint32_t m = __reduce_max_sync(kAll, best);
        if (m == 0) break;
        uint32_t winner;
        if (!keyed) {
            winner = __ffs(__ballot_sync(kAll, best == m)) - 1;
        } else {
            const float mf = unorder_f32(m);
            const uint32_t bar = fabsf(mf) < INFINITY ? order_f32(mf - 2.f * (score_error + 0x1p-22f * fabsf(mf))) : m;
            const uint32_t near = __ballot_sync(kAll, best >= bar);
            if (__popc(near) == 1 && !__any_sync(kAll, second >= bar)) {
                winner = __ffs(near) - 1;
            } else {
                need_sum64();
                uint64_t exact = 0;
                uint32_t exact_i = 0;
#pragma unroll 1
                for (uint32_t i = 0; i < n; ++i) {
                    uint32_t k = 0;
#pragma unroll
                    for (int s = 0; s < kPerLane; ++s) k = uint32_t(s) == i ? key[s] : k;
                    if (k == 0 || k < bar) continue;
                    float l, b;
                    load_logit(p, row, first + i, l, b);
                    const uint64_t o = order_f64(key_f64(p, stats, l, b));
                    if (o > exact) { exact = o; exact_i = i; }
                }
                const uint32_t high = uint32_t(exact >> 32), low = uint32_t(exact);
                const uint32_t top_high = __reduce_max_sync(kAll, high);
                const uint32_t top_low = __reduce_max_sync(kAll, high == top_high ? low : 0u);
                winner = __ffs(__ballot_sync(kAll, exact != 0 && high == top_high && low == top_low)) - 1;
                if (lane == winner) best_i = exact_i;
            }
        }
        const uint32_t e = __shfl_sync(kAll, first + best_i, winner);
        if (lane == j) chosen = int(e);
        if (lane == winner) {
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) key[i] = uint32_t(i) == best_i ? 0u : key[i];
            rescan();
        }
    }

    // Weights: lane j has the j-th choice.  Renormalised scores are ratios, so they are
    // taken relative to the largest chosen one and no sum underflows:
    // sigmoid(l) = e^l / (1 + e^l) = e^m * (e^(l-m) / (1 + e^l)), m = min(0, largest l).
    float l = -INFINITY;
    if (chosen >= 0) {
        float b;
        load_logit(p, row, chosen, l, b);
    }
    float weight = 0.f;
    if (p.renormalize) {
        float peak = l;
#pragma unroll
        for (uint32_t d = 16; d > 0; d >>= 1) peak = fmaxf(peak, __shfl_xor_sync(kAll, peak, d));
        if (chosen >= 0) {
            if (!p.sigmoid) weight = expf(l - peak);
            else if (l > 0.f) weight = 1.f / (1.f + expf(-l));
            else weight = expf(l - fminf(peak, 0.f)) / (1.f + expf(l));
        }
        float sum = weight;
#pragma unroll
        for (uint32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
        if (chosen >= 0) weight /= sum;
    } else if (chosen >= 0) {
        weight = score(l);
    }
    if (lane < p.topk) {
        const uint64_t at = static_cast<uint64_t>(t) * p.topk + lane;
        p.topk_idx[at] = chosen;
        p.topk_weights[at] = weight * p.scale;
    }
}

}  // namespace gcmoe
