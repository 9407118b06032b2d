// Router logits: logits[t][e] = sum_k x[t][k] * W[e][k], BF16 activations, f32 sums and result.
//
// W is kept as P BF16 planes [P][E][H] whose sum is the router's weight: one plane for a BF16
// weight, three for an f32 weight (8 + 8 + 8 significant bits), so that every product is an
// exact product of BF16 values and the result has the accuracy of f32 sums.
//
// A CTA takes kExperts experts and kTokens tokens; its threads run over K side by side and
// their sums are added in a fixed order (no atomics, no dependence on the grid).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_common.cuh"
#include "ptx.cuh"
#include "rms_norm.cuh"

namespace gcmoe {

constexpr uint32_t kLogitsThreads = 256;

struct LogitsParams {
    const __nv_bfloat16* x;       // [T][H]
    const __nv_bfloat16* weight;  // [P][E][H]
    float* out;                   // [T][E]
    uint64_t x_stride;            // elements between rows
    uint32_t num_tokens, num_experts, hidden;
};

template <int kTokens, int kExperts, int kPlanes>
__global__ void __launch_bounds__(kLogitsThreads) logits_fma_kernel(const LogitsParams p) {
    constexpr int kSums = kTokens * kExperts;
    __shared__ float partial[kLogitsThreads / 32][kSums];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t e0 = blockIdx.x * kExperts, t0 = blockIdx.y * kTokens;
    const uint32_t chunks = p.hidden / 8;
    ptx::launch_dependents();
    ptx::grid_dependency_wait();

    float acc[kTokens][kExperts] = {};
    for (uint32_t c = tid; c < chunks; c += kLogitsThreads) {
        uint4 xr[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            xr[i] = make_uint4(0, 0, 0, 0);
            if (t0 + i < p.num_tokens) xr[i] = __ldg(reinterpret_cast<const uint4*>(p.x + (t0 + i) * p.x_stride) + c);
        }
#pragma unroll
        for (int e = 0; e < kExperts; ++e) {
            uint4 wr[kPlanes];
#pragma unroll
            for (int q = 0; q < kPlanes; ++q) {
                wr[q] = make_uint4(0, 0, 0, 0);
                if (e0 + e < p.num_experts)
                    wr[q] = __ldg(reinterpret_cast<const uint4*>(p.weight + (uint64_t(q) * p.num_experts + e0 + e) * p.hidden) + c);
            }
            float w[8];
            unpack_bf16x8(wr[0], w);
            if constexpr (kPlanes == 3) {              // exact: the planes are the bits of one f32
                float mid[8], low[8];
                unpack_bf16x8(wr[1], mid);
                unpack_bf16x8(wr[2], low);
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] += mid[j] + low[j];
            }
#pragma unroll
            for (int i = 0; i < kTokens; ++i) {
                float v[8];
                unpack_bf16x8(xr[i], v);
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[i][e] = fmaf(v[j], w[j], acc[i][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kTokens; ++i)
#pragma unroll
        for (int e = 0; e < kExperts; ++e) {
            float v = acc[i][e];
#pragma unroll
            for (uint32_t d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
            if (lane == 0) partial[warp][i * kExperts + e] = v;
        }
    __syncthreads();
    if (tid < kSums) {
        const uint32_t t = t0 + tid / kExperts, e = e0 + tid % kExperts;
        float v = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kLogitsThreads / 32; ++w) v += partial[w][tid];
        if (t < p.num_tokens && e < p.num_experts) p.out[static_cast<uint64_t>(t) * p.num_experts + e] = v;
    }
}

}  // namespace gcmoe
