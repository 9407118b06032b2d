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
// The order is that of the keys computed in 64 bits, whatever the sums' order in 32: a row
// is chosen by f32 keys with a bound on their error, and is in doubt where two neighbours in
// the order lie within that bound of each other (exact ties among them).
//
// One warp per token; each of a group's lanes holds consecutive experts in registers.  Keys
// are integers that order like the floats (0 = not eligible) whose lowest bits are replaced
// by the expert's place in its lane, so that equal keys go to the lower expert and a
// minimum or maximum moves key and expert together: a lane's list is sorted with two
// instructions per comparison, and a round of the selection is one redux.max, a ballot and the
// winner's next key from shared memory.  The replaced bits count as part of the keys' error.
//
// A row in doubt ranks its picks, and the few experts that may belong among them, by f64
// keys, one per lane; only where more than 32 are in doubt are the choices made again one by
// one (measured: with all rows in doubt made again, 16384 x 256 took 19.8 us, and 16.6 so).
//
// Bound by the integer pipe for many tokens (16384 x 256 in 8 groups, top 8: 15.1 us,
// 780 instructions a row, 340 of them there) and by launch and latency for few (1 x 256: 2.6 us); the bytes
// (E logits in, 12 k out) are small beside both.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cfloat>
#include <cstring>
#include <stdint.h>
#include <type_traits>

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
    uint32_t lanes_log2;          // lanes of a group, a power of two; lanes * num_groups <= 32
    uint32_t per_lane;            // experts of a lane: ceil(group_size / lanes)
    uint32_t sigmoid, group_by_max, renormalize;
    float scale;
};

// Integers in the order of the floats; -0 and +0 are the same, and no float maps to 0.
__device__ __forceinline__ uint32_t order_f32(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unorder_f32(uint32_t u) {
    return __uint_as_float(u ^ (u & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t order_f64(double v) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return b ^ (b >> 63 ? 0xffffffffffffffffull : 0x8000000000000000ull);
}

template <typename T>
__device__ __forceinline__ float logit_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else return static_cast<float>(v);
}
__device__ __forceinline__ float min_nan(float a, float b) {          // NaN if either is
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// NaN stays NaN, +inf becomes the largest finite float.
__device__ __forceinline__ float clean_logit(float l) { return min_nan(l, FLT_MAX); }

// A row's logit, its bias, and whether the expert can be chosen at all (false for NaN too).
template <typename T>
__device__ __forceinline__ bool load_logit(const RouteParams& p, uint64_t row, uint32_t e, float& l, float& b) {
    l = clean_logit(logit_f32(static_cast<const T*>(p.logits)[row + e]));
    b = p.bias != nullptr ? p.bias[e] : 0.f;
    return l > -INFINITY && b > -INFINITY;
}

// kCount consecutive values at an address aligned to 16 bytes, or to all of them.
template <int kCount, typename T>
__device__ __forceinline__ void load_run(const T* from, float (&v)[kCount]) {
    constexpr int kBytes = kCount * int(sizeof(T));
    using Vec = std::conditional_t<kBytes % 16 == 0, uint4, std::conditional_t<kBytes == 8, uint2, uint32_t>>;
    static_assert(kBytes % sizeof(Vec) == 0, "a run is whole vectors");
    constexpr int kPer = int(sizeof(Vec) / sizeof(T));
#pragma unroll
    for (int i = 0; i < kCount / kPer; ++i) {
        const Vec raw = __ldca(reinterpret_cast<const Vec*>(from) + i);
        T part[kPer];
        memcpy(part, &raw, sizeof(Vec));
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[i * kPer + j] = logit_f32(part[j]);
    }
}

// For keys: approximate exponential (2^(-l log2 e)) and reciprocal; the bound on the error
// below covers them.
__device__ __forceinline__ float sigmoid_approx(float l) {
    float z;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(z) : "f"(l * -1.44269504f));
    return ptx::rcp_approx_ftz(1.f + z);
}
__device__ __forceinline__ float sigmoid_f32(float l) {
    const float z = expf(-fabsf(l));
    return (l >= 0.f ? 1.f : z) / (1.f + z);
}

// Softmax statistics of the row: exact maximum, sum in 32 bits.
struct RowStats {
    float top, sum;
};

template <typename T>
__device__ double row_sum_f64(const RouteParams& p, uint64_t row, uint32_t first, uint32_t n, float top) {
    double sum = 0.0;
    for (uint32_t i = 0; i < n; ++i) {
        float l, b;
        if (load_logit<T>(p, row, first + i, l, b)) sum += exp(double(l) - double(top));
    }
#pragma unroll 1
    for (uint32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
}

// The score plus bias in 64 bits.
__device__ __forceinline__ double key_f64(const RouteParams& p, float top, double sum, float l, float b) {
    if (p.sigmoid) return 1.0 / (1.0 + exp(-double(l))) + double(b);
    return exp(double(l) - double(top)) / sum + double(b);
}

// Rank of this lane's group by f64 values (scores: sums of two or the largest).
template <typename T>
__device__ __noinline__ uint32_t group_rank_f64(const RouteParams& p, uint64_t row, uint32_t first, uint32_t n, uint32_t group,
                                                float top, bool by_sum) {
    constexpr uint32_t kAll = 0xffffffffu;
    const bool scored = p.bias != nullptr || by_sum;
    const double sum = scored && !p.sigmoid ? row_sum_f64<T>(p, row, first, n, top) : 1.0;
    double b1 = -INFINITY, b2 = -INFINITY;
    for (uint32_t i = 0; i < n; ++i) {
        float l, b;
        if (!load_logit<T>(p, row, first + i, l, b)) continue;
        const double m = scored ? key_f64(p, top, sum, l, b) : double(l);
        b2 = fmax(b2, fmin(b1, m));
        b1 = fmax(b1, m);
    }
    for (uint32_t d = (1u << p.lanes_log2) >> 1; d > 0; d >>= 1) {
        const double o1 = __shfl_xor_sync(kAll, b1, d), o2 = __shfl_xor_sync(kAll, b2, d);
        b2 = fmax(fmin(b1, o1), fmax(b2, o2));
        b1 = fmax(b1, o1);
    }
    const double mine = by_sum && b2 > -INFINITY ? b1 + b2 : b1;
    uint32_t rank = 0;
    for (uint32_t o = 0; o < p.num_groups; ++o) {
        const double v = __shfl_sync(kAll, mine, o << p.lanes_log2);
        rank += v > mine || (v == mine && o < group);
    }
    return rank;
}

// A choice's key in 64 bits, as an integer: the logit itself without a bias.
__device__ __forceinline__ uint64_t choice_key(const RouteParams& p, float top, double sum, float l, float b) {
    return order_f64(p.bias != nullptr ? key_f64(p, top, sum, l, b) : double(l));
}

// The row's choices by f64 keys, one after the other, for rows with more experts in doubt
// than a warp has lanes (most of a row alike): lane j returns the j-th expert, or -1.
template <typename T>
__device__ __noinline__ int choose_f64(const RouteParams& p, uint64_t row, uint32_t first, uint32_t n, bool eligible, float top,
                                       double sum) {
    constexpr uint32_t kAll = 0xffffffffu;
    uint64_t taken = eligible ? 0ull : ~0ull;                          // n is at most 64
    int chosen = -1;
    for (uint32_t j = 0; j < p.topk; ++j) {
        uint64_t best = 0;
        uint32_t at = 0;
        for (uint32_t i = 0; i < n; ++i) {
            float l, b;
            if ((taken >> i & 1) || !load_logit<T>(p, row, first + i, l, b)) continue;
            const uint64_t key = choice_key(p, top, sum, l, b);
            if (key > best) { best = key; at = i; }                    // equal keys: the first
        }
        const uint32_t high = uint32_t(best >> 32), low = uint32_t(best);
        const uint32_t top_high = __reduce_max_sync(kAll, high);
        if (top_high == 0) break;                                      // no float orders below 2^32
        const uint32_t top_low = __reduce_max_sync(kAll, high == top_high ? low : 0u);
        const uint32_t winner = __ffs(__ballot_sync(kAll, high == top_high && low == top_low)) - 1;
        const uint32_t e = __shfl_sync(kAll, first + at, winner);
        if (threadIdx.x % 32 == j) chosen = int(e);
        if (threadIdx.x % 32 == winner) taken |= 1ull << at;
    }
    return chosen;
}

// Batcher's odd-even merge sort of a lane's list, largest first.
template <int kCount>
__device__ __forceinline__ void sort_descending(uint32_t (&v)[kCount]) {
#pragma unroll
    for (int p = 1; p < kCount; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int i = 0; i + k < kCount; ++i)
                if (i >= k % p && (i - k % p) / k % 2 == 0 && i / (2 * p) == (i + k) / (2 * p)) {
                    const uint32_t x = v[i], y = v[i + k];
                    v[i] = max(x, y);
                    v[i + k] = min(x, y);
                }
}

// Whether the order of two neighbours is in doubt: keys a >= b, of which the lowest bits
// (`mask`) are not the float's, each off by at most `error` and the rounding of a sum, 2^-24
// of its size (the difference taken here rounds once more).
__device__ __forceinline__ bool in_doubt(uint32_t a, uint32_t b, uint32_t mask, float error) {
    const float low = unorder_f32(a & ~mask), high = unorder_f32(b | mask);
    return b != 0 && !(low - high > 2.f * error + 0x1p-22f * fmaxf(fabsf(low), fabsf(high)));   // NaN: in doubt
}

// kFull: every lane of a group has kPerLane experts, in rows aligned for vector loads
// (16384 x 256 in 15.1 us, element by element 17.5; 1 x 256 2.58 and 2.65).
template <typename T, int kPerLane, bool kFull>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const __grid_constant__ RouteParams p) {
    constexpr uint32_t kAll = 0xffffffffu;
    constexpr bool kSorted = kPerLane <= 16;
    constexpr uint32_t kPlace = kPerLane - 1u;        // bits of a key that hold the place; kPerLane is a power of two
    __shared__ uint32_t lists[kRouteWarps][kSorted ? kPerLane - 1 : 1][32], ranked[kRouteWarps][32];
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t t = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    ptx::launch_dependents();
    ptx::grid_dependency_wait();
    if (t >= p.num_tokens) return;                    // whole warps

    const uint64_t row = t * p.logits_stride;
    const uint32_t group = lane >> p.lanes_log2, sub = lane & ((1u << p.lanes_log2) - 1u);
    const uint32_t begin = sub * p.per_lane;
    const uint32_t n = group < p.num_groups && begin < p.group_size ? min(p.per_lane, p.group_size - begin) : 0u;
    const uint32_t first = group * p.group_size + begin;
    const bool keyed = p.bias != nullptr;             // keys are scores, not logits

    // Logits, then keys.  -inf or NaN: not eligible; a comparison with -inf tells both.
    float value[kPerLane], bias[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) { value[i] = -INFINITY; bias[i] = 0.f; }
    if constexpr (kFull) {
        if (n != 0) {
            load_run<kPerLane>(static_cast<const T*>(p.logits) + row + first, value);
            if (keyed) load_run<kPerLane>(p.bias + first, bias);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (uint32_t(i) < n) {
                value[i] = logit_f32(static_cast<const T*>(p.logits)[row + first + i]);
                if (keyed) bias[i] = p.bias[first + i];
            }
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) value[i] = clean_logit(value[i]);

    const bool by_sum = p.num_groups > 1 && !p.group_by_max;
    RowStats stats = {0.f, 1.f};
    if (!p.sigmoid && (keyed || by_sum || !p.renormalize)) {
        // masked experts have no part in the softmax; an empty row keeps top = 0
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (bias[i] > -INFINITY) top = fmaxf(top, value[i]);       // fmaxf passes over NaN
        top = unorder_f32(__reduce_max_sync(kAll, order_f32(top)));
        if (top > -INFINITY) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i)
                if (value[i] > -INFINITY && bias[i] > -INFINITY) sum += expf(value[i] - top);
#pragma unroll
            for (uint32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
            stats.top = top;
            stats.sum = sum;
        }
    }
    // Bound on the f32 error of a score.  Sigmoid, below one: the approximate exponential is
    // off by 2 + 1.2 |l| steps of 2^-23, times s (1 - s) at most 0.65 steps; the sum and the
    // reciprocal add 1.5: 2.15 steps.  Softmax, below inv_sum: the sum's roundings (2048 terms
    // at most, 69 of them one after the other) and the exponential's, below 2^-17 of it.
    const float inv_sum = 1.f / stats.sum;
    const float score_error = p.sigmoid ? 0x1.2p-22f : 0x1p-17f * inv_sum;
    // l * 0 makes the score of a masked logit NaN and leaves the others alone
    auto score = [&](float l) { return fmaf(l, 0.f, p.sigmoid ? sigmoid_approx(l) : expf(l - stats.top) * inv_sum); };
    if (keyed) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) value[i] = score(value[i]) + bias[i];
    }
    constexpr bool kShort = sizeof(T) == 2;           // as f32, the low 13 bits of every logit are alike

    bool eligible = true;                             // this lane's group is among the best
    if (p.num_groups > 1) {
        const bool scored = keyed || by_sum;          // the groups' values come from scores
        float a1 = -INFINITY, a2 = -INFINITY;         // the two largest members of the lane, then of the group
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const float m = !keyed && by_sum ? score(value[i]) : value[i];
            a2 = fmaxf(a2, min_nan(a1, m));           // fmaxf passes over NaN
            a1 = fmaxf(a1, m);
        }
        for (uint32_t d = (1u << p.lanes_log2) >> 1; d > 0; d >>= 1) {
            const float o1 = __shfl_xor_sync(kAll, a1, d), o2 = __shfl_xor_sync(kAll, a2, d);
            a2 = fmaxf(fminf(a1, o1), fmaxf(a2, o2));
            a1 = fmaxf(a1, o1);
        }
        const bool two = by_sum && a2 > -INFINITY;
        const float mine = two ? a1 + a2 : a1;        // -inf: nothing left in the group
        // the group's place in the low bits; a group without members orders last, by place
        const uint32_t packed = group < p.num_groups ? (order_f32(mine) & ~31u) | (31u - group) : 0u;
        uint32_t left = packed, border = 0;
        for (uint32_t r = 0; r < p.topk_groups; ++r) {
            border = __reduce_max_sync(kAll, left);
            if (left == border) left = 0;
        }
        const uint32_t next = __reduce_max_sync(kAll, left);
        eligible = packed >= border;
        const bool empty = group < p.num_groups && mine == -INFINITY;
        bool doubt = (border ^ next) < 32u && !(kShort && !scored);    // alike but for the place
        if (scored) {
            const float size = fabsf(mine) < INFINITY ? fabsf(a1) + (two ? fabsf(a2) : 0.f) : 0.f;
            const float error = 2.f * score_error + 0x1p-22f * __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(size)));
            doubt = in_doubt(border, next, 31u, error);
        }
        // among groups without members the place decides: nothing is in doubt
        if (doubt && !(__all_sync(kAll, left == 0 || empty)))
            eligible = group_rank_f64<T>(p, row, first, n, group, stats.top, by_sum) < p.topk_groups;
    }

    // The lane's keys.  A lane outside the best groups adds -inf; fmaxf makes NaN -inf; + 0 makes -0 +0.
    uint32_t list[kPerLane];
    const float in_group = eligible ? 0.f : -INFINITY;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
        list[i] = (order_f32(fmaxf(value[i] + in_group, -INFINITY)) & ~kPlace) | (kPlace - uint32_t(i));
    // Up to 16 experts are sorted.  The two best are in registers, what follows in shared
    // memory: a choice then moves one key up, whatever the list's length.
    // A scan of the list in each round takes 17.7 us instead of 15.1 for 16384 x 256, 2.83
    // instead of 2.58 for 1 x 256.
    uint32_t best = list[0], second = 0, down = 0;    // down: where the next key lies
    if constexpr (kSorted) {
        sort_descending(list);
        best = list[0];
        second = list[1];
        uint32_t* const rest = &lists[threadIdx.x >> 5][0][lane];
#pragma unroll
        for (int i = 2; i < kPerLane; ++i) rest[(i - 2) * 32] = list[i];
        rest[(kPerLane - 2) * 32] = 0;                // below every key, for whoever asks further
    }
    auto lane_best = [&]() {
        if constexpr (!kSorted) {
            best = list[0];
#pragma unroll
            for (int i = 1; i < kPerLane; ++i) best = max(best, list[i]);
        }
        return best;
    };
    constexpr uint32_t kNone = 0x007fffffu;           // order_f32(-inf), whose low bits are all set
    uint2 pick = make_uint2(0u, 0u);                  // lane j: the j-th choice's key and its lane
    // A round: the lane with the largest key m (of equal ones, the lower lane has the lower
    // expert) gives it to lane `place` and passes on to its next.
    auto round = [&](uint32_t place, uint32_t m) {
        const uint32_t winner = __ffs(__ballot_sync(kAll, (best | kPlace) == m)) - 1;
        const uint32_t key = __shfl_sync(kAll, best, winner);
        if (lane == place) pick = make_uint2(key, winner);
        if constexpr (kSorted) {
            if (lane == winner) {
                best = second;
                second = lists[threadIdx.x >> 5][down][lane];
                down = min(down + 1, uint32_t(kPerLane - 2));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) list[i] = lane == winner && list[i] == key ? 0u : list[i];
        }
    };
    uint32_t count = 0;                               // choices made
    uint32_t m = __reduce_max_sync(kAll, lane_best() | kPlace);
    while (count < p.topk && m > kNone) {
        round(count++, m);
        m = __reduce_max_sync(kAll, lane_best() | kPlace);
    }
    const uint32_t last = m > kNone ? m : 0u;         // the best key that is left
    auto order_in_doubt = [&](uint32_t a, uint32_t b) {
        return keyed ? in_doubt(a, b, kPlace, score_error) : !kShort && (a ^ b) <= kPlace;
    };
    auto expert_of = [&](uint2 pick) {                // owner's group, its part of the group, place
        return (pick.y >> p.lanes_log2) * p.group_size + (pick.y & ((1u << p.lanes_log2) - 1u)) * p.per_lane + kPlace -
               (pick.x & kPlace);
    };
    const uint32_t after = __shfl_down_sync(kAll, pick.x, 1);
    int chosen = lane < count ? int(expert_of(pick)) : -1;
    if (__any_sync(kAll, lane < count && order_in_doubt(pick.x, lane + 1 == p.topk ? last : after))) {
        // Exact keys for the picks and for what else may belong among them.
        const double sum = keyed && !p.sigmoid ? row_sum_f64<T>(p, row, first, n, stats.top) : 1.0;
        const uint32_t border = __shfl_sync(kAll, pick.x, p.topk - 1);   // the last pick, if there are that many
        bool many = false;
        while (count >= p.topk && m > kNone && order_in_doubt(border, m)) {
            many = count == 32;
            if (many) break;
            round(count++, m);
            m = __reduce_max_sync(kAll, lane_best() | kPlace);
        }
        if (many) {
            chosen = choose_f64<T>(p, row, first, n, eligible, stats.top, sum);
        } else {
            uint64_t key = 0;
            uint32_t e = 0xffffffffu;
            if (lane < count) {
                float l, b;
                e = expert_of(pick);
                load_logit<T>(p, row, e, l, b);
                key = choice_key(p, stats.top, sum, l, b);
            }
            uint32_t rank = 0;
            for (uint32_t o = 0; o < count; ++o) {
                const uint64_t k = __shfl_sync(kAll, key, o);
                const uint32_t other = __shfl_sync(kAll, e, o);
                rank += k > key || (k == key && other < e);
            }
            uint32_t* const order = ranked[threadIdx.x >> 5];
            if (lane < count) order[rank] = e;
            __syncwarp();
            chosen = lane < min(count, p.topk) ? int(order[lane]) : -1;
        }
    }

    // Weights: lane j has the j-th choice.  Renormalised scores are ratios, so they are
    // taken relative to the largest chosen one and no sum underflows:
    // sigmoid(l) = e^l / (1 + e^l) = e^m * (e^(l-m) / (1 + e^l)), m = min(0, largest l).
    float l = -INFINITY;
    if (chosen >= 0) l = clean_logit(logit_f32(static_cast<const T*>(p.logits)[row + chosen]));
    float weight = 0.f;
    if (p.renormalize) {
        const float peak = unorder_f32(__reduce_max_sync(kAll, order_f32(l)));
        if (p.sigmoid) {
            const float z = expf(-fabsf(l));          // -inf (no choice): 0
            weight = l > 0.f ? 1.f : peak > 0.f ? z : expf(l - peak);
            weight = __fdividef(weight, 1.f + z);
        } else {
            weight = expf(l - peak);
        }
        if (chosen < 0) weight = 0.f;
        float sum = weight;
#pragma unroll
        for (uint32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
        if (chosen >= 0) weight = __fdividef(weight, sum);
    } else if (chosen >= 0) {
        weight = p.sigmoid ? sigmoid_f32(l) : expf(l - stats.top) / stats.sum;
    }
    if (lane < p.topk) {
        const uint64_t out = static_cast<uint64_t>(t) * p.topk + lane;
        p.topk_idx[out] = chosen;
        p.topk_weights[out] = weight * p.scale;
    }
}

}  // namespace gcmoe
